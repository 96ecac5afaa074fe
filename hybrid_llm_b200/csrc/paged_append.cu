// New tokens into a paged key-value cache: RMS norm of every query and key
// head, rotary positions, keys and values stored in their pages, in one pass.
//
//   n(x)  = x / sqrt(mean(x^2) + eps) * w                 (w given)
//   r(x)  = (a cos t - b sin t, b cos t + a sin t), t = position * inv_freq[i]
//           over the pairs (a, b) = (x[i], x[i + half]) or (x[2i], x[2i + 1])
//
// Token t of sequence b (cu_q[b] <= t < cu_q[b + 1]) has position
// lengths[b] - cu_q[b + 1] + t: the sequence's last tokens are the new ones.
// The angle is formed and reduced to [-pi, pi] in 64 bits (a product rounded
// to 32 bits is off by 0.06 rad at position 10^6), its sine and cosine and
// everything else in 32, with one rounding at the store.
//
// Bound by its bytes, or by latency for a few tokens.  A warp takes some heads
// of one token, 16 bytes per lane: its rows are asked for first, and the
// sequence's lookups and the angles (two per lane, handed round by shuffles, the
// same for every head) run while they travel; no barrier, no shared memory.
#include "paged.cuh"
#include "tma_host.h"

namespace llmyb {
namespace {

constexpr int kThreads = 256;  // 8 warps that know nothing of each other

struct AppendArgs {
  const uint16_t *q, *k, *v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  uint16_t* q_out;
  int64_t o_tok, o_head;
  uint16_t *k_pages, *v_pages;
  PagedPool pool;
  const int32_t* cu_q;  // null: one token per sequence
  int32_t n_tokens, q_heads;
  const float *q_norm, *k_norm;
  float eps;
  const float* inv_freq;
  int32_t half, interleaved;
  int32_t* dev_status;
};

// How a token's heads are dealt to warps: `rounds` rounds of 32 / (DH / 8) heads
// each, every warp with heads of one kind (queries, keys or values).
struct Parts {
  int q, kv;  // warps for the queries, for the keys and for the values
};

template <typename T, int DH, int kRounds>
__global__ void __launch_bounds__(kThreads, 4) paged_append_kernel(AppendArgs a, Parts parts) {
  constexpr int kLanes = DH / 8, kHeads = 32 / kLanes;
  const int lane = threadIdx.x & 31, l = lane % kLanes;
  // eight tokens' part of one kind per CTA; the parts of a token are neighbours
  const unsigned per = parts.q + 2 * parts.kv;
  const int tok = static_cast<int>(blockIdx.x / per) * (kThreads / 32) + (threadIdx.x >> 5);
  if (tok >= a.n_tokens) return;
  int part = static_cast<int>(blockIdx.x % per);
  const int kind = part < parts.q ? 0 : part < parts.q + parts.kv ? 1 : 2;
  part -= kind == 0 ? 0 : kind == 1 ? parts.q : parts.q + parts.kv;
  const int heads = kind == 0 ? a.q_heads : a.pool.kv_heads;
  const int h0 = part * (kRounds * kHeads) + lane / kLanes;
  const uint16_t* const src = (kind == 0   ? a.q + tok * a.q_tok
                               : kind == 1 ? a.k + tok * a.k_tok
                                           : a.v + tok * a.v_tok) + 8 * l;
  const int64_t src_head = kind == 0 ? a.q_head : kind == 1 ? a.k_head : a.v_head;
  uint4 raw[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int h = h0 + i * kHeads;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (h < heads) raw[i] = __ldcs(reinterpret_cast<const uint4*>(src + h * src_head));
  }
  int b = tok, pos;
  if (a.cu_q != nullptr) {
    const int begin = a.cu_q[0], end = a.cu_q[a.pool.batch];
    // the last b with cu_q[b] <= tok, 32 candidates at a time
    b = 0;
    for (int n = a.pool.batch; n > 1;) {
      const int step = (n + 31) / 32, at = (lane + 1) * step;
      const bool below = at < n && a.cu_q[b + at] <= tok;
      const int skip = __popc(__ballot_sync(0xffffffffu, below)) * step;
      b += skip;
      n = min(step, n - skip);
    }
    if (tok < begin || tok >= end) return;  // rows of no sequence
    pos = a.pool.lengths[b] - a.cu_q[b + 1] + tok;
  } else {
    pos = a.pool.lengths[b] - 1;
  }
  uint16_t* dst = a.q_out + tok * a.o_tok;
  int64_t dst_head = a.o_head;
  if (kind != 0) {
    if (pos < 0) return;  // a slot without a token
    const int page_i = pos >> a.pool.page_shift;
    int page = -1;
    if (page_i < a.pool.table_width) page = a.pool.table[b * a.pool.table_stride + page_i];
    if (page < 0 || page >= a.pool.num_pages) {
      if (lane == 0) report_status(a.dev_status, LLMYB_EINVAL);
      return;
    }
    dst = (kind == 1 ? a.k_pages : a.v_pages) + static_cast<int64_t>(page) * a.pool.page_stride +
          (pos & ((1 << a.pool.page_shift) - 1)) * a.pool.row_stride;
    dst_head = a.pool.head_stride;
  }
  dst += 8 * l;
  const float* const norm = kind == 0 ? a.q_norm : a.k_norm;
  // a query without a position is zero whatever norm and angle would make of it
  const bool copy = kind == 2 || pos < 0 || (norm == nullptr && a.half == 0);

  // x'_k = r (x_k u_k + y_k v_k), y the other member of the pair and r the
  // inverse RMS: u = weight cos, v = -+ the other's weight sin, the same for
  // every head of this warp
  float u[8], v[8];
  const int d = a.half / 8;  // lanes between the two members of a half-split pair
  const bool second = l >= d && l < 2 * d;
  const int other = l < d ? l + d : second ? l - d : l;
  const bool turns = a.half > 0 && 8 * l < 2 * a.half;
  if (!copy) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      u[k] = norm ? norm[8 * l + k] : 1.f;
      v[k] = 0.f;
    }
    if (a.half > 0) {
      float c[2] = {1.f, 1.f}, s[2] = {0.f, 0.f};  // of pairs 2 lane and 2 lane + 1
      if (2 * lane < a.half) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          constexpr double kTwoPi = 6.283185307179586476925286766559;
          const double t = static_cast<double>(pos) * static_cast<double>(a.inv_freq[2 * lane + i]);
          // 2^-21 of absolute error on [-pi, pi]
          __sincosf(static_cast<float>(t - rint(t * (1.0 / kTwoPi)) * kTwoPi), &s[i], &c[i]);
        }
      }
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int from = (4 * l + i) >> 1 & 31;
          const float cc = __shfl_sync(0xffffffffu, c[i & 1], from);
          const float ss = __shfl_sync(0xffffffffu, s[i & 1], from);
          if (turns) {
            const float w0 = u[2 * i], w1 = u[2 * i + 1];
            u[2 * i] = w0 * cc, v[2 * i] = -w1 * ss;
            u[2 * i + 1] = w1 * cc, v[2 * i + 1] = w0 * ss;
          }
        }
      } else {
        const int first = 8 * (second ? l - d : l);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int from = (first + k) >> 1 & 31;
          const float cc = __shfl_sync(0xffffffffu, c[k & 1], from);
          const float ss = __shfl_sync(0xffffffffu, s[k & 1], from);
          if (turns) {
            v[k] = (second ? ss : -ss) * (norm ? norm[8 * other + k] : 1.f);
            u[k] *= cc;
          }
        }
      }
    }
  }
  const int peer = lane - l + other;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int h = h0 + i * kHeads;
    if (part * (kRounds * kHeads) + i * kHeads >= heads) break;
    uint4 o = raw[i];
    if (pos < 0) o = make_uint4(0, 0, 0, 0);
    if (!copy) {
      uint4 p = o;  // the pairs' other members
      if (!a.interleaved && a.half > 0) {
        p.x = __shfl_sync(0xffffffffu, o.x, peer), p.y = __shfl_sync(0xffffffffu, o.y, peer);
        p.z = __shfl_sync(0xffffffffu, o.z, peer), p.w = __shfl_sync(0xffffffffu, o.w, peer);
      }
      const float2 x[4] = {Elem<T>::unpack(o.x), Elem<T>::unpack(o.y), Elem<T>::unpack(o.z),
                           Elem<T>::unpack(o.w)};
      float r = 1.f;
      if (norm != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) ss = fmaf(x[k].x, x[k].x, fmaf(x[k].y, x[k].y, ss));
#pragma unroll
        for (int k = kLanes / 2; k > 0; k >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, k);
        r = rsqrtf(ss * (1.f / DH) + a.eps);
      }
      float2 z[4];
      if (!turns) {  // by itself: zero times an infinity is none
#pragma unroll
        for (int k = 0; k < 4; ++k) z[k] = make_float2(x[k].x * u[2 * k], x[k].y * u[2 * k + 1]);
      } else if (a.interleaved) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          z[k] = make_float2(fmaf(x[k].x, u[2 * k], x[k].y * v[2 * k]),
                             fmaf(x[k].y, u[2 * k + 1], x[k].x * v[2 * k + 1]));
      } else {
        const float2 y[4] = {Elem<T>::unpack(p.x), Elem<T>::unpack(p.y), Elem<T>::unpack(p.z),
                             Elem<T>::unpack(p.w)};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          z[k] = make_float2(fmaf(x[k].x, u[2 * k], y[k].x * v[2 * k]),
                             fmaf(x[k].y, u[2 * k + 1], y[k].y * v[2 * k + 1]));
      }
      o = make_uint4(Elem<T>::pack(z[0].x * r, z[0].y * r), Elem<T>::pack(z[1].x * r, z[1].y * r),
                     Elem<T>::pack(z[2].x * r, z[2].y * r), Elem<T>::pack(z[3].x * r, z[3].y * r));
    }
    if (h < heads) *reinterpret_cast<uint4*>(dst + h * dst_head) = o;
  }
}

// Rounds per warp: one where that many warps do not fill the GPU's 64 per SM
// (a token's latency counts), else eight, so that a token's lookups and angles
// serve several heads: 14117 tokens of 16 + 2 x 16 heads, 347 MB, take 70 us
// in a graph of calls (0.76 of the copy rate; 74 us as single calls), with 72 %
// of the issue slots busy.  Four rounds took 85 us where eight took 77; a CTA
// per token with the angles in shared memory, 129 us.
template <typename T, int DH, int kRounds>
void launch(const AppendArgs& a, cudaStream_t s) {
  constexpr int kHeads = kRounds * (256 / DH);
  const Parts p = {(a.q_heads + kHeads - 1) / kHeads, (a.pool.kv_heads + kHeads - 1) / kHeads};
  const int64_t ctas = ceil_div(a.n_tokens, kThreads / 32) * (p.q + 2 * p.kv);
  paged_append_kernel<T, DH, kRounds><<<static_cast<unsigned>(ctas), kThreads, 0, s>>>(a, p);
}
template <typename T, int DH>
void launch(const AppendArgs& a, cudaStream_t s) {
  const int64_t rounds = ceil_div(a.q_heads + 2 * a.pool.kv_heads, 256 / DH);
  if (a.n_tokens * rounds <= 64ll * num_sms()) launch<T, DH, 1>(a, s);
  else launch<T, DH, 8>(a, s);
}

}  // namespace
}  // namespace llmyb

using namespace llmyb;

LLMYB_API int32_t llmyb_paged_append(const llmyb_paged_args* x, void* stream) {
  const int32_t st = paged_check(x);
  if (st) return st;
  if (x->rope_half < 0 || !(x->eps >= 0.f)) return LLMYB_EINVAL;
  if (x->n_tokens == 0 || x->batch == 0) return LLMYB_OK;
  if (!x->k || !x->v || (x->rope_half > 0 && !x->inv_freq) || (!x->cu_q && x->n_tokens != x->batch))
    return LLMYB_EINVAL;
  if (x->rope_half % 8 != 0 || 2 * x->rope_half > x->head_dim ||
      !paged_aligned(x->k, x->k_token_stride, x->k_head_stride) ||
      !paged_aligned(x->v, x->v_token_stride, x->v_head_stride) || !paged_aligned(x->q_norm) ||
      !paged_aligned(x->k_norm))
    return LLMYB_EUNSUPPORTED;
  AppendArgs a;
  a.q = static_cast<const uint16_t*>(x->q), a.k = static_cast<const uint16_t*>(x->k);
  a.v = static_cast<const uint16_t*>(x->v);
  a.q_tok = x->q_token_stride, a.q_head = x->q_head_stride;
  a.k_tok = x->k_token_stride, a.k_head = x->k_head_stride;
  a.v_tok = x->v_token_stride, a.v_head = x->v_head_stride;
  a.q_out = static_cast<uint16_t*>(x->out);
  a.o_tok = x->out_token_stride, a.o_head = x->out_head_stride;
  a.k_pages = static_cast<uint16_t*>(x->k_pages), a.v_pages = static_cast<uint16_t*>(x->v_pages);
  a.pool = paged_pool(x);
  a.cu_q = x->cu_q, a.n_tokens = x->n_tokens, a.q_heads = x->q_heads;
  a.q_norm = x->q_norm, a.k_norm = x->k_norm, a.eps = x->eps;
  a.inv_freq = x->inv_freq, a.half = x->rope_half, a.interleaved = x->interleaved;
  a.dev_status = x->dev_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x->fp16) {
    if (x->head_dim == 64) launch<__half, 64>(a, s);
    else launch<__half, 128>(a, s);
  } else {
    if (x->head_dim == 64) launch<__nv_bfloat16, 64>(a, s);
    else launch<__nv_bfloat16, 128>(a, s);
  }
  count_launch();
  return launch_status();
}
