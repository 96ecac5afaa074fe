// Shared by the paged key-value cache operators (append, decode, prefill): the
// cache's layout, the two 16-bit element types and the score transforms.
//
// A cache is two pools of pages, keys and values, [page][kv head][row][head
// dim] with free strides over page, head and row (a [page][row][head][dim]
// pool is the same with other strides).  table[b][i] names the page that holds
// positions [i * page_size, (i + 1) * page_size) of sequence b; lengths[b]
// counts its positions, the ones appended for the current call included.
#pragma once

#include <cuda_fp16.h>
#include "common.cuh"
#include "../../include/llmyb.h"

namespace llmyb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct PagedPool {
  int64_t page_stride, head_stride, row_stride;  // elements
  int32_t num_pages, page_shift;                 // page_size = 1 << page_shift
  const int32_t* table;
  int64_t table_stride;
  int32_t table_width;  // pages per sequence at most
  const int32_t* lengths;
  int32_t batch, kv_heads;

  __device__ __forceinline__ int length(int b) const {
    return max(0, min(lengths[b], table_width << page_shift));
  }
};

// 16-bit element types: pack two fp32 values, unpack two, 1.0 of the type.
template <typename T>
struct Elem;

template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return unpack_bf16x2(v); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

template <>
struct Elem<__half> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&p);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    __half2 p = *reinterpret_cast<__half2*>(&v);
    return __half22float2(p);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// tanh x = 1 - 2 / (1 + e^2x): absolute error below 2^-21 (one exp2 and one
// reciprocal of the special-function unit; the tanh instruction's 2^-11 would
// move a score capped at 50 by 0.02, a probability by 2 %).
__device__ __forceinline__ float tanh_exp(float x) {
  return 1.f - 2.f * fast_rcp(1.f + fast_exp2(x * (2.f * kLog2e)));
}

// log2 of the row's unnormalised weight sum -> natural log-sum-exp
__device__ __forceinline__ float lse_of(float m, float l) {
  return l > 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
}

inline int page_shift_of(int page_size) {
  switch (page_size) {
    case 16: return 4;
    case 32: return 5;
    case 64: return 6;
    case 128: return 7;
    case 256: return 8;
    default: return -1;
  }
}

inline bool paged_aligned(const void* p, int64_t a = 0, int64_t b = 0) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && a % 8 == 0 && b % 8 == 0;
}

// What the three calls check alike: LLMYB_OK, or why not.  Call it before
// anything else; a call without tokens or sequences needs no pointers.
inline int32_t paged_check(const llmyb_paged_args* a) {
  if (!a || a->n_tokens < 0 || a->batch < 0 || a->q_heads <= 0 || a->kv_heads <= 0 ||
      a->num_pages < 0 || a->table_width < 0)
    return LLMYB_EINVAL;
  if (a->n_tokens == 0 || a->batch == 0) return LLMYB_OK;
  if (!a->q || !a->k_pages || !a->v_pages || !a->table || !a->lengths || !a->out ||
      a->num_pages == 0)
    return LLMYB_EINVAL;
  const int shift = page_shift_of(a->page_size);
  if (shift < 0 || (a->head_dim != 64 && a->head_dim != 128) ||
      a->table_width > (1 << 30) >> shift ||
      !paged_aligned(a->q, a->q_token_stride, a->q_head_stride) ||
      !paged_aligned(a->out, a->out_token_stride, a->out_head_stride) ||
      !paged_aligned(a->k_pages, a->page_stride, a->head_stride) ||
      !paged_aligned(a->v_pages, a->row_stride))
    return LLMYB_EUNSUPPORTED;
  return LLMYB_OK;
}

// Further for the attention calls.
inline int32_t paged_check_scores(const llmyb_paged_args* a) {
  if (a->q_heads % a->kv_heads != 0 || a->window < 0 || !(a->scale > 0.f) || !(a->softcap >= 0.f))
    return LLMYB_EINVAL;
  return LLMYB_OK;
}

inline PagedPool paged_pool(const llmyb_paged_args* a) {
  return {a->page_stride, a->head_stride, a->row_stride, a->num_pages,
          page_shift_of(a->page_size), a->table, a->table_stride, a->table_width, a->lengths,
          a->batch, a->kv_heads};
}

}  // namespace llmyb
