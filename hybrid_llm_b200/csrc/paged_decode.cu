// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale q.k_j;  s_j = cap tanh(s_j / cap);  s_j -= slope_h (p - j)
//   out = sum_j softmax(s)_j v_j over the visible j <= p = length - 1,
//   p - j < window.  A sequence of length 0 gives zeros.
//
// Bound by the cache's bytes: every key and value row is read once for all the
// query heads that share it (16 rows of an m16n8k16 product; larger groups in
// chunks of 16).  The batch's keys form one flat list of (sequence, kv head,
// tile) which is cut into equal shares, one per WARP of a grid that just fills
// the GPU, so lengths may be as uneven as they like and one long sequence uses
// every SM.  A warp is a worker of its own: its ring of cp.async stages runs
// across the boundaries of sequences, it keeps the running maximum and sum of
// the softmax and 16 x DH outputs in registers, and no barrier ties it to the
// other warps.  A sequence-head that one worker holds whole is written at
// once; the pieces of the others go to scratch (unnormalised sum, maximum,
// weight sum, fp32) and a second launch joins them, in a fixed order.  Short
// caches go without: a CTA per sequence and kv head, its four warps joined in
// shared memory.
#include <algorithm>

#include "mma.cuh"
#include "paged.cuh"
#include "tma_host.h"

namespace llmyb {
namespace {

constexpr int kWarps = 4;        // workers per CTA
constexpr int kCtasPerSm = 2;
constexpr int kStages = 3;
constexpr int kStageBytes = 8192;  // keys 4 KB, values 4 KB
constexpr int kSmem = kWarps * kStages * kStageBytes;

struct DecodeArgs {
  const uint16_t* q;
  int64_t q_tok, q_head;
  const uint16_t *k_pages, *v_pages;
  PagedPool pool;
  int32_t group, chunks, rows;  // heads per kv head, chunks of them, heads per chunk at most
  int32_t q_heads, window, workers;
  int32_t whole;  // a CTA per (sequence, kv head, chunk), joined in shared memory
  float scale, softcap;
  const float* slopes;
  uint16_t* out;
  int64_t o_tok, o_head;
  float* lse;  // [batch, q_heads] or null
  float* part_o;   // [workers * 2][rows][DH]
  float2* part_ml; // [workers * 2][rows]
  int32_t* dev_status;
};

// Visible tiles of sequence b: the first one and how many (at least one).
template <int KT>
__device__ __forceinline__ void tiles_of(const DecodeArgs& a, int b, int& len, int& lo, int& first,
                                         int& count) {
  len = a.pool.length(b);
  lo = a.window > 0 ? max(0, len - a.window) : 0;
  first = lo / KT;
  count = max(1, (len + KT - 1) / KT - first);
}

// Tiles of the whole batch for one (kv head, chunk), by one warp.
template <int KT>
__device__ __forceinline__ int64_t total_tiles(const DecodeArgs& a) {
  const int lane = threadIdx.x & 31;
  int64_t sum = 0;
  for (int b = lane; b < a.pool.batch; b += 32) {
    int len, lo, first, count;
    tiles_of<KT>(a, b, len, lo, first, count);
    sum += count;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

__device__ __forceinline__ int64_t share_of(int64_t tiles, int workers) {
  return (tiles + workers - 1) / workers;
}

// A position in the flat list of tiles.
struct Cursor {
  int b, hc;               // sequence, kv head * chunks + chunk
  int tile, count, first;  // of this sequence
  int len, lo;

  template <int KT>
  __device__ __forceinline__ void enter(const DecodeArgs& a) {
    tiles_of<KT>(a, b, len, lo, first, count);
  }
  // false: the list is at its end
  template <int KT>
  __device__ __forceinline__ void next(const DecodeArgs& a) {
    if (++tile < count) return;
    tile = 0;
    if (++hc < a.pool.kv_heads * a.chunks) return;
    hc = 0;
    if (++b < a.pool.batch) enter<KT>(a);
  }
};

// Sequence whose tiles (times hcs) hold flat position `at`, and the tiles
// before it; by one warp.
template <int KT>
__device__ __forceinline__ int find_sequence(const DecodeArgs& a, int64_t at, int hcs,
                                             int64_t& before) {
  const int lane = threadIdx.x & 31;
  before = 0;
  for (int b0 = 0;; b0 += 32) {
    int64_t mine = 0;
    if (b0 + lane < a.pool.batch) {
      int len, lo, first, count;
      tiles_of<KT>(a, b0 + lane, len, lo, first, count);
      mine = static_cast<int64_t>(count) * hcs;
    }
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, before + inc > at);
    if (hit != 0) {
      const int l = __ffs(hit) - 1;
      before += __shfl_sync(0xffffffffu, inc - mine, l);
      return b0 + l;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
    if (b0 + 32 >= a.pool.batch) return a.pool.batch;
  }
}

template <typename T, int DH>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm) paged_decode_kernel(DecodeArgs a) {
  constexpr int KT = 2048 / DH;   // keys per tile: 16 or 32
  constexpr int kPieces = KT / 16;
  constexpr int kCh = DH / 8;     // 16-byte pieces per row
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int worker = blockIdx.x * kWarps + warp;
  pdl_trigger();
  const int hcs = a.pool.kv_heads * a.chunks;
  uint8_t* ring = smem + warp * kStages * kStageBytes;
  Cursor ld;  // where the loads are
  int n_load;
  if (a.whole) {  // a quarter of one segment's tiles
    ld.b = blockIdx.x / hcs;
    ld.hc = blockIdx.x % hcs;
    ld.enter<KT>(a);
    ld.tile = warp * ld.count / kWarps;
    n_load = (warp + 1) * ld.count / kWarps - ld.tile;
  } else {
    const int64_t tiles = total_tiles<KT>(a) * hcs;
    const int64_t share = share_of(tiles, a.workers);
    const int64_t t0 = worker * share, t1 = min(tiles, t0 + share);
    if (t0 >= t1) return;
    n_load = static_cast<int>(t1 - t0);
    int64_t before;
    ld.b = find_sequence<KT>(a, t0, hcs, before);
    ld.enter<KT>(a);
    const int64_t r = t0 - before;
    ld.hc = static_cast<int>(r / ld.count);
    ld.tile = static_cast<int>(r % ld.count);
  }
  Cursor cu = ld;  // where the products are
  int n_left = n_load;
  int page[kPieces];  // of the next tile to load
  auto look_up = [&]() {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int key = (ld.first + ld.tile) * KT + 16 * i;
      page[i] = -1;
      if (key < ld.len && key + 15 >= ld.lo)
        page[i] = a.pool.table[ld.b * a.pool.table_stride + (key >> a.pool.page_shift)];
    }
  };
  look_up();
  auto load = [&](int stage) {
    if (n_load > 0) {
      uint8_t* kd = ring + stage * kStageBytes;
      const int kvh = ld.hc / a.chunks;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int key0 = (ld.first + ld.tile) * KT + 16 * i;
        const bool held = key0 < ld.len && key0 + 15 >= ld.lo;
        bool ok = held && page[i] >= 0 && page[i] < a.pool.num_pages;
        if (held && !ok && lane == 0) report_status(a.dev_status, LLMYB_EINVAL);
        const int64_t base =
            ok ? static_cast<int64_t>(page[i]) * a.pool.page_stride + kvh * a.pool.head_stride +
                     (key0 & ((1 << a.pool.page_shift) - 1)) * a.pool.row_stride
               : 0;
#pragma unroll
        for (int c = 0; c < 16 * kCh / 32; ++c) {
          const int x = c * 32 + lane;
          const int row = x / kCh, col = x % kCh;
          // rows outside the sequence are not read: they may hold anything,
          // and a zero weight does not cancel an infinity
          const bool in = ok && key0 + row >= ld.lo && key0 + row < ld.len;
          const int64_t src = in ? base + row * a.pool.row_stride + 8 * col : 0;
          const uint32_t dst = (16 * i + row) * (2 * DH) + ((col ^ (row & 7)) << 4);
          mma::cp_async16(kd + dst, a.k_pages + src, in);
          mma::cp_async16(kd + 4096 + dst, a.v_pages + src, in);
        }
      }
      ld.next<KT>(a);
      if (--n_load > 0) look_up();
    }
    mma::cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load(s);

  uint32_t qf[DH / 16][4];
  float o[DH / 8][4];
  float m[2], l[2], slope[2];
  int rows = 0;
  const int r0 = lane >> 2, c0 = 2 * (lane & 3);
  auto begin = [&]() {  // the queries of the segment at `cu`
    const int head0 = (cu.hc / a.chunks) * a.group + (cu.hc % a.chunks) * 16;
    rows = min(16, a.group - (cu.hc % a.chunks) * 16);
    const uint16_t* q = a.q + cu.b * a.q_tok + head0 * a.q_head;
#pragma unroll
    for (int ks = 0; ks < DH / 16; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + (i & 1) * 8;
        qf[ks][i] = r < rows ? *reinterpret_cast<const uint32_t*>(q + r * a.q_head + 16 * ks + c0 +
                                                                  (i >> 1) * 8)
                             : 0u;
      }
#pragma unroll
    for (int i = 0; i < DH / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
      slope[i] = a.slopes && r0 + 8 * i < rows ? a.slopes[head0 + r0 + 8 * i] * kLog2e : 0.f;
    }
  };
  begin();
  const float sc = a.scale * kLog2e, cap = a.softcap * kLog2e;
  const float cap_in = a.softcap > 0.f ? 2.f * a.scale / a.softcap : 0.f;
  bool whole_start = !a.whole && cu.tile == 0;  // this worker holds the segment's first tile
  bool first_segment = true;
  int stage = 0;

  while (n_left > 0) {
    mma::cp_async_wait<kStages - 2>();
    __syncwarp();
    load(stage == 0 ? kStages - 1 : stage - 1);  // the stage read one tile ago
    const uint8_t* kd = ring + stage * kStageBytes;
    const uint8_t* vd = kd + 4096;
    stage = stage == kStages - 1 ? 0 : stage + 1;

    // scores of 16 rows x KT keys
    float s[KT / 8][4];
#pragma unroll
    for (int n = 0; n < KT / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < DH / 16; ++ks)
#pragma unroll
      for (int n2 = 0; n2 < KT / 16; ++n2) {
        uint32_t bk[4];
        const int row = 16 * n2 + (lane & 7) + (lane >> 4) * 8;
        const int col = 2 * ks + ((lane >> 3) & 1);
        mma::ldsm_x4(bk, kd + row * (2 * DH) + ((col ^ (row & 7)) << 4));
        Elem<T>::mma(s[2 * n2], qf[ks], bk[0], bk[1]);
        Elem<T>::mma(s[2 * n2 + 1], qf[ks], bk[2], bk[3]);
      }
    const int key0 = (cu.first + cu.tile) * KT;
    // distance of the lane's first key: formed in whole numbers, positions pass 2^24
    const float d0 = static_cast<float>(cu.len - 1 - key0 - c0);
    if (a.softcap > 0.f) {
      uint32_t big = 0u;  // bit 30: a score past the cap
#pragma unroll
      for (int n = 0; n < KT / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] *= cap_in;
          big |= __float_as_uint(s[n][e]);
        }
      // they are rare; a tile without takes the short form, to the same results
      if (__builtin_expect(__any_sync(0xffffffffu, big & 0x40000000u), 0)) {
#pragma unroll
        for (int n = 0; n < KT / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float2 t = split2(tanh_half_exp2(make2(s[n][e], s[n][e + 1])));
            s[n][e] = t.x, s[n][e + 1] = t.y;
          }
      } else {
#pragma unroll
        for (int n = 0; n < KT / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float2 t = split2(tanh_half_poly2(make2(s[n][e], s[n][e + 1])));
            s[n][e] = t.x, s[n][e + 1] = t.y;
          }
      }
    }
    const float to2 = a.softcap > 0.f ? cap : sc;  // to scores in base 2
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < KT / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + 8 * n + c0 + (e & 1);
        float x = s[n][e] * to2;
        if (a.slopes) x = fmaf(-slope[e >> 1], d0 - static_cast<float>(8 * n + (e & 1)), x);
        x = key >= cu.lo && key < cu.len ? x : -INFINITY;
        s[n][e] = x;
        top[e >> 1] = fmaxf(top[e >> 1], x);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2)) - Elem<T>::kDecodeUp;
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float t = fmaxf(m[i], top[i]);
        f[i] = t == m[i] ? 1.f : fast_exp2(m[i] - t);
        m[i] = t;
        l[i] *= f[i];
      }
#pragma unroll
      for (int n = 0; n < DH / 8; ++n) {
        o[n][0] *= f[0], o[n][1] *= f[0];
        o[n][2] *= f[1], o[n][3] *= f[1];
      }
    }
    const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
    for (int n = 0; n < KT / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = fast_exp2(s[n][e] - base[e >> 1]);
        l[e >> 1] += s[n][e];
      }
    // Weights rounded to the cache's type, the operand that the tensor cores take:
    // each off by at most half a step, unbiased, so the output's own rounding
    // stays the larger part (errors against 64 bits 0.0022 of the output's size,
    // 0.0017 with fp32 weights).  Their sum takes them unrounded.
#pragma unroll
    for (int ks = 0; ks < KT / 16; ++ks) {
      const uint32_t p[4] = {Elem<T>::pack(s[2 * ks][0], s[2 * ks][1]),
                             Elem<T>::pack(s[2 * ks][2], s[2 * ks][3]),
                             Elem<T>::pack(s[2 * ks + 1][0], s[2 * ks + 1][1]),
                             Elem<T>::pack(s[2 * ks + 1][2], s[2 * ks + 1][3])};
#pragma unroll
      for (int d2 = 0; d2 < DH / 16; ++d2) {
        uint32_t bv[4];
        const int row = 16 * ks + (lane & 7) + ((lane >> 3) & 1) * 8;
        const int col = 2 * d2 + (lane >> 4);
        mma::ldsm_x4_t(bv, vd + row * (2 * DH) + ((col ^ (row & 7)) << 4));
        Elem<T>::mma(o[2 * d2], p, bv[0], bv[1]);
        Elem<T>::mma(o[2 * d2 + 1], p, bv[2], bv[3]);
      }
    }
    --n_left;
    const bool seg_end = cu.tile + 1 == cu.count;
    if (seg_end || n_left == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      }
      if (a.whole) {
        // (joined below)
      } else if (seg_end && whole_start) {
        const int head0 = (cu.hc / a.chunks) * a.group + (cu.hc % a.chunks) * 16;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = r0 + 8 * i;
          if (r >= rows) continue;
          const float inv = inv_of(l[i]);
          uint16_t* dst = a.out + cu.b * a.o_tok + (head0 + r) * a.o_head + c0;
#pragma unroll
          for (int n = 0; n < DH / 8; ++n)
            *reinterpret_cast<uint32_t*>(dst + 8 * n) =
                Elem<T>::pack(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
          if (a.lse && (lane & 3) == 0)
            a.lse[static_cast<int64_t>(cu.b) * a.q_heads + head0 + r] = lse_of(m[i], l[i]);
        }
      } else {
        const int slot = 2 * worker + (first_segment ? 0 : 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = r0 + 8 * i;
          if (r >= rows) continue;
          const int64_t at = static_cast<int64_t>(slot) * a.rows + r;
          float* dst = a.part_o + at * DH + c0;
#pragma unroll
          for (int n = 0; n < DH / 8; ++n)
            *reinterpret_cast<float2*>(dst + 8 * n) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
          if ((lane & 3) == 0) a.part_ml[at] = make_float2(m[i], l[i]);
        }
      }
      if (n_left == 0) break;
      cu.next<KT>(a);
      begin();
      whole_start = true;
      first_segment = false;
    } else {
      ++cu.tile;
    }
  }
  mma::cp_async_wait<0>();
  if (!a.whole) return;
  // the warps' pieces, through their rings
  float* const piece = reinterpret_cast<float*>(ring);
  float2* const piece_ml = reinterpret_cast<float2*>(ring + 16 * DH * 4);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = r0 + 8 * i;
#pragma unroll
    for (int n = 0; n < DH / 8; ++n)
      *reinterpret_cast<float2*>(piece + r * DH + 8 * n + c0) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
    if ((lane & 3) == 0) piece_ml[r] = make_float2(m[i], l[i]);
  }
  __syncthreads();
  const int b = blockIdx.x / hcs, hc = blockIdx.x % hcs;
  const int head0 = (hc / a.chunks) * a.group + (hc % a.chunks) * 16;
  for (int x = threadIdx.x; x < rows * (DH / 4); x += kWarps * 32) {
    const int r = x / (DH / 4), c = x % (DH / 4);
    float2 ml[kWarps];
    float4 p[kWarps];
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const uint8_t* const from = smem + w * kStages * kStageBytes;
      ml[w] = reinterpret_cast<const float2*>(from + 16 * DH * 4)[r];
      p[w] = reinterpret_cast<const float4*>(from)[r * (DH / 4) + c];
      top = fmaxf(top, ml[w].x);
    }
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = fast_exp2(ml[w].x - base);
      sum = fmaf(ml[w].y, f, sum);
      y.x = fmaf(p[w].x, f, y.x), y.y = fmaf(p[w].y, f, y.y);
      y.z = fmaf(p[w].z, f, y.z), y.w = fmaf(p[w].w, f, y.w);
    }
    const float inv = inv_of(sum);
    *reinterpret_cast<uint2*>(a.out + b * a.o_tok + (head0 + r) * a.o_head + 4 * c) =
        make_uint2(Elem<T>::pack(y.x * inv, y.y * inv), Elem<T>::pack(y.z * inv, y.w * inv));
    if (a.lse && c == 0) a.lse[static_cast<int64_t>(b) * a.q_heads + head0 + r] = lse_of(top, sum);
  }
}

// Joins the pieces of the sequence-heads that several workers share: one CTA
// per (sequence, kv head, chunk, row), NT threads.
template <typename T, int DH, int NT>
__global__ void __launch_bounds__(NT) paged_decode_join_kernel(DecodeArgs a) {
  constexpr int KT = 2048 / DH;
  constexpr int kVec = DH / 4;                  // threads per part's row
  constexpr int kLanes = NT / kVec;   // parts read side by side
  __shared__ float4 s_o[kLanes][kVec];
  __shared__ float s_red[NT / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.x % a.rows;
  const int seg = blockIdx.x / a.rows;
  const int hcs = a.pool.kv_heads * a.chunks;
  const int b = seg / hcs, hc = seg % hcs;
  if (r >= min(16, a.group - (hc % a.chunks) * 16)) {
    pdl_wait();
    return;
  }
  // tiles before this sequence and in the whole batch (every warp for itself)
  int64_t before = 0, tiles = 0;
  int count = 1;
  for (int i = lane; i < a.pool.batch; i += 32) {
    int len, lo, first, n;
    tiles_of<KT>(a, i, len, lo, first, n);
    tiles += n;
    if (i < b) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  {
    int len, lo, first;
    tiles_of<KT>(a, b, len, lo, first, count);
  }
  const int64_t share = share_of(tiles * hcs, a.workers);
  const int64_t t0 = before * hcs + static_cast<int64_t>(hc) * count, t1 = t0 + count;
  const int w0 = static_cast<int>(t0 / share), w1 = static_cast<int>((t1 - 1) / share);
  // every CTA waits, those without work too: the launch must not be over
  // before the one that it depends on
  pdl_wait();
  if (w0 == w1) return;
  const int head = (hc / a.chunks) * a.group + (hc % a.chunks) * 16 + r;
  auto at = [&](int w) -> int64_t {
    return (2ll * w + (w == w0 && t0 > w0 * share ? 1 : 0)) * a.rows + r;
  };
  float m = -INFINITY;
  for (int w = w0 + threadIdx.x; w <= w1; w += NT) m = fmaxf(m, a.part_ml[at(w)].x);
  m = warp_max(m);
  if (lane == 0) s_red[warp] = m;
  __syncthreads();
  m = s_red[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) m = fmaxf(m, s_red[i]);
  const float base = m == -INFINITY ? 0.f : m;
  const int v = threadIdx.x % kVec, p = threadIdx.x / kVec;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 5
  for (int w = w0 + p; w <= w1; w += kLanes) {
    const float2 ml = a.part_ml[at(w)];
    const float4 x = *reinterpret_cast<const float4*>(a.part_o + at(w) * DH + 4 * v);
    const float f = fast_exp2(ml.x - base);
    l = fmaf(ml.y, f, l);
    o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y);
    o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
  }
  s_o[p][v] = o;
  __shared__ float s_l[kLanes];
  if (v == 0) s_l[p] = l;
  __syncthreads();
  if (p != 0) return;
  l = s_l[0];
#pragma unroll
  for (int i = 1; i < kLanes; ++i) {
    const float4 x = s_o[i][v];
    o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
    l += s_l[i];
  }
  const float inv = inv_of(l);
  uint16_t* dst = a.out + b * a.o_tok + head * a.o_head + 4 * v;
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(Elem<T>::pack(o.x * inv, o.y * inv), Elem<T>::pack(o.z * inv, o.w * inv));
  if (a.lse && v == 0) a.lse[static_cast<int64_t>(b) * a.q_heads + head] = lse_of(m, l);
}

// One CTA per sequence and kv head instead of equal shares, by what the table
// can hold: where that is a few tiles (the second launch costs more: 300 keys
// of 8 heads of 64, 5.8 us against 6.3 and one launch less for the host), and
// where there are CTAs enough to even lengths out (64 x 4 heads of 128 with
// 1024 keys: 25.1 us against 30.8; with few CTAs uneven lengths would leave SMs idle).
bool whole_segments(int64_t segments, int table_width, int page_size, int head_dim) {
  const int64_t tiles = static_cast<int64_t>(table_width) * page_size / (2048 / head_dim);
  return segments <= 0x7fffffff && (tiles <= 16 || (tiles <= 64 && segments >= 4 * num_sms()));
}

int worker_count() { return num_sms() * kCtasPerSm * kWarps; }

template <typename T, int DH>
int32_t launch(const DecodeArgs& a, cudaStream_t s) {
  int32_t st = ensure_smem(paged_decode_kernel<T, DH>, kSmem);
  if (st) return st;
  const int64_t segments = static_cast<int64_t>(a.pool.batch) * a.pool.kv_heads * a.chunks;
  paged_decode_kernel<T, DH>
      <<<static_cast<unsigned>(a.whole ? segments : a.workers / kWarps), kWarps * 32, kSmem, s>>>(a);
  st = launch_status();
  if (st || a.whole) {
    count_launch();
    return st;
  }
  // Pieces per row: with few rows there are many (one sequence, 4 kv heads:
  // 296), which 128 threads read one after another in 29 us, 1024 in 7.
  const dim3 grid(static_cast<unsigned>(segments * a.rows));
  const cudaError_t e =
      a.workers > 16 * segments
          ? launch_pdl(paged_decode_join_kernel<T, DH, 1024>, grid, dim3(1024), 0, s, a)
          : launch_pdl(paged_decode_join_kernel<T, DH, 128>, grid, dim3(128), 0, s, a);
  count_launch(2);
  return e == cudaSuccess ? launch_status() : static_cast<int32_t>(e);
}

}  // namespace
}  // namespace llmyb

using namespace llmyb;

LLMYB_API int64_t llmyb_paged_decode_scratch_bytes(int32_t q_heads, int32_t kv_heads,
                                                   int32_t head_dim) {
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || head_dim <= 0) return -1;
  const int64_t rows = std::min(16, q_heads / kv_heads);
  return static_cast<int64_t>(worker_count()) * 2 * rows * (head_dim + 2) * 4;
}

LLMYB_API int32_t llmyb_paged_decode(const llmyb_paged_args* x, void* stream) {
  int32_t st = paged_check(x);
  if (st) return st;
  st = paged_check_scores(x);
  if (st) return st;
  if (x->n_tokens != x->batch) return LLMYB_EINVAL;
  if (x->batch == 0) return LLMYB_OK;
  if (!x->scratch) return LLMYB_EINVAL;
  if (!paged_aligned(x->scratch)) return LLMYB_EUNSUPPORTED;
  DecodeArgs a;
  a.q = static_cast<const uint16_t*>(x->q), a.q_tok = x->q_token_stride, a.q_head = x->q_head_stride;
  a.k_pages = static_cast<const uint16_t*>(x->k_pages);
  a.v_pages = static_cast<const uint16_t*>(x->v_pages);
  a.pool = paged_pool(x);
  a.group = x->q_heads / x->kv_heads;
  a.chunks = (a.group + 15) / 16;
  a.rows = std::min(16, a.group);
  a.q_heads = x->q_heads, a.window = x->window, a.workers = worker_count();
  a.whole = whole_segments(static_cast<int64_t>(x->batch) * x->kv_heads * a.chunks, x->table_width,
                           x->page_size, x->head_dim);
  a.scale = x->scale, a.softcap = x->softcap, a.slopes = x->slopes;
  a.out = static_cast<uint16_t*>(x->out);
  a.o_tok = x->out_token_stride, a.o_head = x->out_head_stride;
  a.lse = x->lse;
  a.part_o = static_cast<float*>(x->scratch);
  a.part_ml = reinterpret_cast<float2*>(a.part_o +
                                        static_cast<int64_t>(a.workers) * 2 * a.rows * x->head_dim);
  a.dev_status = x->dev_status;
  if (static_cast<int64_t>(x->batch) * x->kv_heads * a.chunks * a.rows > 0x7fffffffll)
    return LLMYB_EUNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x->fp16) return x->head_dim == 64 ? launch<__half, 64>(a, s) : launch<__half, 128>(a, s);
  return x->head_dim == 64 ? launch<__nv_bfloat16, 64>(a, s) : launch<__nv_bfloat16, 128>(a, s);
}
