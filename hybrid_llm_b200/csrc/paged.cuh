// Shared by the paged key-value cache operators (append, decode, prefill): the
// cache's layout, the two 16-bit element types and the score transforms.
//
// A cache is two pools of pages, keys and values, [page][kv head][row][head
// dim] with free strides over page, head and row (a [page][row][head][dim]
// pool is the same with other strides).  table[b][i] names the page that holds
// positions [i * page_size, (i + 1) * page_size) of sequence b; lengths[b]
// counts its positions, the ones appended for the current call included.
#pragma once

#include <cfloat>

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

// 16-bit element types: pack two fp32 values, unpack two.  Softmax weights are
// rounded to the type for the second product, in which fp16 holds nothing below
// 2^-25: there the largest weight is 2^kDecodeUp, or in the prompt kernel
// 2^kPrefillUp, which needs the rest for maxima that rise later, so that the many
// small weights of a long cache are kept (with a largest weight of 1, 40,000 keys
// 25 bits below the best one vanished from the output, 0.1 % of it, but not from
// the weights' sum).  bf16 has the exponents of fp32.
template <typename T>
struct Elem;

template <>
struct Elem<__nv_bfloat16> {
  static constexpr float kDecodeUp = 0.f, kPrefillUp = 0.f, kMostWeight = 16384.f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return unpack_bf16x2(v); }
  // acc, or NaN where v or acc is not finite
  static __device__ __forceinline__ uint32_t probe(uint32_t v, uint32_t acc) {
    __nv_bfloat162 r = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&v), __nv_bfloat162{}, *reinterpret_cast<__nv_bfloat162*>(&acc));
    return *reinterpret_cast<uint32_t*>(&r);
  }
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
  static constexpr float kDecodeUp = 12.f, kPrefillUp = 4.f;
  static constexpr float kMostWeight = 57344.f;  // below the type's largest, 65504
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&p);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    __half2 p = *reinterpret_cast<__half2*>(&v);
    return __half22float2(p);
  }
  // acc, or NaN where v or acc is not finite
  static __device__ __forceinline__ uint32_t probe(uint32_t v, uint32_t acc) {
    __half2 r = __hfma2(*reinterpret_cast<__half2*>(&v), __half2{}, *reinterpret_cast<__half2*>(&acc));
    return *reinterpret_cast<uint32_t*>(&r);
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

// natural log-sum-exp from the base-2 maximum and the weight sum (0: no key)
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// 1 / l, and 0 for a row without keys; a NaN stays one
__device__ __forceinline__ float inv_of(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Two fp32 values in one 64-bit register: one issue slot for two operations.
__device__ __forceinline__ uint64_t make2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ float2 split2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// tanh x ~ x P(x^2) for |x| < 1: minimax fit of the RELATIVE error, 5.9e-7
// (7.0e-7 with fp32 rounding), so that a score far below the cap keeps its digits
// however large the cap is.
constexpr double kTanh0 = 0.9999994135992633, kTanh1 = -0.3332904237853046,
                 kTanh2 = 0.1328143388070316, kTanh3 = -0.05160567400105457,
                 kTanh4 = 0.016743115062558066, kTanh5 = -0.003067060326103062;

// tanh of half of each value, |y| < 2, by that with the factor 1/2 in the
// coefficients: "out of range" is one bit of the argument (2^1 and above,
// infinities and NaN have bit 30 set).
__device__ __forceinline__ uint64_t tanh_half_poly2(uint64_t y) {
  const uint64_t z = mul2(y, y);
  auto c = [](double v) { return make2(static_cast<float>(v), static_cast<float>(v)); };
  uint64_t p = fma2(z, c(kTanh5 / 2048), c(kTanh4 / 512));
  p = fma2(z, p, c(kTanh3 / 128));
  p = fma2(z, p, c(kTanh2 / 32));
  p = fma2(z, p, c(kTanh1 / 8));
  p = fma2(z, p, c(kTanh0 / 2));
  return mul2(p, y);
}

// The same for any y: from 2 on 1 - 2 / (1 + e^y), whose ABSOLUTE error of 2^-22
// (one exp2 and one reciprocal of the special-function unit) would be multiplied
// by the cap for small y (0.012 of a score at a cap of 1e5); the tanh
// instruction's 2^-11 would move a score capped at 50 by 0.02, a probability by 2 %.
__device__ __forceinline__ uint64_t tanh_half_exp2(uint64_t y) {
  const float2 near = split2(tanh_half_poly2(y)), v = split2(y);
  auto of = [](float v, float near) {
    const float far = 1.f - 2.f * fast_rcp(1.f + fast_exp2(v * kLog2e));
    return fabsf(v) < 2.f ? near : far;  // far: a NaN too
  };
  return make2(of(v.x, near.x), of(v.y, near.y));
}

// The same for any y with one special function for two values: from 2 on, with
// x = y / 2 clamped to 7, x P(x^2) / Q(x^2), minimax fit of the absolute error
// (1.1e-6 with fp32 rounding; 1.7e-6 where clamped); one reciprocal serves both:
// a/b and c/d are a d / (b d) and c b / (b d), Q in [1, 91].
__device__ __forceinline__ uint64_t tanh_half2(uint64_t y) {
  const float2 near = split2(tanh_half_poly2(y));
  const float2 c = split2(y);
  // the clamp drops a NaN, which would reach the other value by the reciprocal
  const float lo = fminf(fmaxf(0.5f * c.x, -7.f), 7.f), hi = fminf(fmaxf(0.5f * c.y, -7.f), 7.f);
  y = make2(lo, hi);
  const uint64_t z = mul2(y, y);
  uint64_t p = fma2(z, make2(3.9298196e-06f, 3.9298196e-06f), make2(0.0022769469f, 0.0022769469f));
  p = fma2(z, p, make2(0.1230213613f, 0.1230213613f));
  p = fma2(z, p, make2(0.9999956868f, 0.9999956868f));
  p = mul2(p, y);
  uint64_t q = fma2(z, make2(0.00014234632f, 0.00014234632f), make2(0.0210719839f, 0.0210719839f));
  q = fma2(z, q, make2(0.4563398457f, 0.4563398457f));
  q = fma2(z, q, make2(1.f, 1.f));
  const float2 d = split2(q);
  const float r = fast_rcp(d.x * d.y);
  const float2 t = split2(mul2(mul2(p, make2(d.y, d.x)), make2(r, r)));
  auto of = [](float v, float in, float out) { return fabsf(v) < 2.f ? in : v == v ? out : v; };
  return make2(of(c.x, near.x, t.x), of(c.y, near.y, t.y));
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
  // a table without columns has no address: its sequences are all empty
  if (!a->q || !a->k_pages || !a->v_pages || (!a->table && a->table_width > 0) || !a->lengths ||
      !a->out || a->num_pages == 0)
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

// Further for the attention calls.  Scores are formed in base 2 (factors of log2 e,
// below 1.5) and, under a cap,
// as fractions of it: those factors must be numbers of fp32 (a cap so large or
// small that they are not would make every score 0 or NaN).
inline int32_t paged_check_scores(const llmyb_paged_args* a) {
  auto normal = [](float x) { return x >= FLT_MIN && x <= FLT_MAX; };
  if (a->q_heads % a->kv_heads != 0 || a->window < 0 || !normal(a->scale) ||
      !normal(1.5f * a->scale) || !(a->softcap >= 0.f))
    return LLMYB_EINVAL;
  if (a->softcap > 0.f && (!normal(1.5f * a->softcap) || !normal(a->scale / a->softcap) ||
                           !normal(2.f * a->scale / a->softcap)))
    return LLMYB_EINVAL;
  return LLMYB_OK;
}

inline PagedPool paged_pool(const llmyb_paged_args* a) {
  return {a->page_stride, a->head_stride, a->row_stride, a->num_pages,
          page_shift_of(a->page_size), a->table, a->table_stride, a->table_width, a->lengths,
          a->batch, a->kv_heads};
}

}  // namespace llmyb
