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

}  // namespace llmyb
