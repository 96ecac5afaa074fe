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
#include "paged.cuh"

namespace llmyb {
namespace {

constexpr int kThreads = 256;

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

// One CTA per token; DH / 8 lanes per head, 16 bytes each.
template <typename T, int DH>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(AppendArgs a) {
  constexpr int kLanes = DH / 8;
  __shared__ float2 s_rot[DH / 2];  // (cos, sin) of the token's angles
  const int tok = blockIdx.x, tid = threadIdx.x;
  int b = tok, pos;
  if (a.cu_q != nullptr) {
    if (tok >= a.cu_q[a.pool.batch]) return;  // rows behind the last sequence
    int lo = 0, hi = a.pool.batch;            // cu_q[lo] <= tok < cu_q[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_q[mid] <= tok) lo = mid;
      else hi = mid;
    }
    b = lo;
    pos = a.pool.lengths[b] - a.cu_q[b + 1] + tok;
  } else {
    pos = a.pool.lengths[b] - 1;
  }
  if (tid < a.half) {
    constexpr double kTwoPi = 6.283185307179586476925286766559;
    const double t = static_cast<double>(pos) * static_cast<double>(a.inv_freq[tid]);
    float s, c;
    sincosf(static_cast<float>(t - rint(t * (1.0 / kTwoPi)) * kTwoPi), &s, &c);
    s_rot[tid] = make_float2(c, s);
  }
  // the page of this position
  const int page_i = pos >> a.pool.page_shift;
  int page = -1;
  if (pos >= 0) {
    if (page_i < a.pool.table_width) page = a.pool.table[b * a.pool.table_stride + page_i];
    if (page < 0 || page >= a.pool.num_pages) {
      page = -1;
      if (tid == 0) report_status(a.dev_status, LLMYB_EINVAL);
    }
  }
  const int64_t in_page = static_cast<int64_t>(page) * a.pool.page_stride +
                          (pos & ((1 << a.pool.page_shift) - 1)) * a.pool.row_stride;
  __syncthreads();

  const int l = tid % kLanes;
  const int heads = a.q_heads + 2 * a.pool.kv_heads;
  for (int h0 = tid / kLanes; h0 < (heads + kThreads / kLanes - 1) / (kThreads / kLanes) *
                                       (kThreads / kLanes);
       h0 += kThreads / kLanes) {
    const bool live = h0 < heads;
    const int h = min(h0, heads - 1);
    const uint16_t* src;
    uint16_t* dst;
    const float* w = nullptr;
    bool turn = false, store;
    if (h < a.q_heads) {
      src = a.q + tok * a.q_tok + h * a.q_head;
      dst = a.q_out + tok * a.o_tok + h * a.o_head;
      w = a.q_norm;
      turn = true;
      store = live;
    } else if (h < a.q_heads + a.pool.kv_heads) {
      const int g = h - a.q_heads;
      src = a.k + tok * a.k_tok + g * a.k_head;
      dst = a.k_pages + in_page + g * a.pool.head_stride;
      w = a.k_norm;
      turn = true;
      store = live && page >= 0;
    } else {
      const int g = h - a.q_heads - a.pool.kv_heads;
      src = a.v + tok * a.v_tok + g * a.v_head;
      dst = a.v_pages + in_page + g * a.pool.head_stride;
      store = live && page >= 0;
    }
    uint4 raw = *reinterpret_cast<const uint4*>(src + 8 * l);
    if (pos < 0) raw = make_uint4(0, 0, 0, 0);  // a slot without a token: its query is zero
    float x[8];
    {
      const float2 p0 = Elem<T>::unpack(raw.x), p1 = Elem<T>::unpack(raw.y),
                   p2 = Elem<T>::unpack(raw.z), p3 = Elem<T>::unpack(raw.w);
      x[0] = p0.x, x[1] = p0.y, x[2] = p1.x, x[3] = p1.y;
      x[4] = p2.x, x[5] = p2.y, x[6] = p3.x, x[7] = p3.y;
    }
    // the shuffles run in every lane: lane groups of one warp may hold
    // different kinds of heads
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (w != nullptr) {
      const float r = rsqrtf(ss * (1.f / DH) + a.eps);
      const float4 w0 = *reinterpret_cast<const float4*>(w + 8 * l);
      const float4 w1 = *reinterpret_cast<const float4*>(w + 8 * l + 4);
      x[0] *= r * w0.x, x[1] *= r * w0.y, x[2] *= r * w0.z, x[3] *= r * w0.w;
      x[4] *= r * w1.x, x[5] *= r * w1.y, x[6] *= r * w1.z, x[7] *= r * w1.w;
    }
    if (a.half > 0) {
      if (a.interleaved) {
        if (turn && 8 * l < 2 * a.half) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 r = s_rot[4 * l + i];
            const float u = x[2 * i], v = x[2 * i + 1];
            x[2 * i] = u * r.x - v * r.y;
            x[2 * i + 1] = v * r.x + u * r.y;
          }
        }
      } else {
        const int d = a.half / 8;  // lanes between the two members of a pair
        const bool first = l < d, second = l >= d && l < 2 * d;
        const int peer = (threadIdx.x & 31) + (first ? d : second ? -d : 0);
        const int at = first ? 8 * l : second ? 8 * (l - d) : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = __shfl_sync(0xffffffffu, x[i], peer);
          const float2 r = s_rot[at + i];
          if (turn && first) x[i] = x[i] * r.x - y * r.y;
          if (turn && second) x[i] = x[i] * r.x + y * r.y;
        }
      }
    }
    if (store) {
      uint4 o = raw;  // values pass unchanged
      if (turn && (w != nullptr || a.half > 0))
        o = make_uint4(Elem<T>::pack(x[0], x[1]), Elem<T>::pack(x[2], x[3]),
                       Elem<T>::pack(x[4], x[5]), Elem<T>::pack(x[6], x[7]));
      *reinterpret_cast<uint4*>(dst + 8 * l) = o;
    }
  }
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
  const int n = x->n_tokens;
  if (x->fp16) {
    if (x->head_dim == 64) paged_append_kernel<__half, 64><<<n, kThreads, 0, s>>>(a);
    else paged_append_kernel<__half, 128><<<n, kThreads, 0, s>>>(a);
  } else {
    if (x->head_dim == 64) paged_append_kernel<__nv_bfloat16, 64><<<n, kThreads, 0, s>>>(a);
    else paged_append_kernel<__nv_bfloat16, 128><<<n, kThreads, 0, s>>>(a);
  }
  count_launch();
  return launch_status();
}
