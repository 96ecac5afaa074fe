// Attention of several new tokens per sequence (a prompt, or a chunk of one
// behind a cached context) over a paged key-value cache, on 5th-generation
// tensor cores.
//
//   s_ij = scale q_i.k_j;  s = cap tanh(s / cap);  s -= slope_h |i - j|
//   out_i = sum_j softmax_j(s_ij) v_j over the visible j: j <= i, i - j < window,
//   or (instead of a window) j < prefix of the sequence.
// Sequences are packed: tokens cu_q[b] .. cu_q[b + 1) are the last ones of
// sequence b, whose length counts them; a sequence never sees another one.  A
// row that sees no key gives zeros.
//
// A tile is 128 rows = (128 / group) tokens x the group of query heads that
// share a kv head, so keys and values are read once per group and a causal
// tile wastes little on its diagonal.  A unit of work is two such tiles that
// run in turn over the same 128-key blocks, from the diagonal down:
//   warps 0-3, 4-7  softmax of tile 0 / 1 (one row per thread, TMEM lane = row):
//                   scores from TMEM, mask on edge blocks, base-2 online softmax
//                   with a lazily raised maximum (raised only past 2^8, O then
//                   rescaled in TMEM), P in 16 bits over the scores' columns
//   warp 8          TMA: queries once per unit, keys and values page by page in
//                   one ring of 128-key blocks
//   warp 9          MMA: O_t += P_t V then S_t = Q_t K of the next block, for
//                   t = 0, 1: one tile's products run under the other's softmax
// Values of rows outside the sequence (behind its end, or before the window)
// are zeroed in shared memory: they may hold anything, and a zero weight does
// not cancel an infinity.  With few units the key axis of every unit is split
// over several CTAs; their unnormalised fp32 sums are joined by a second launch.
// All waits are bounded; a timeout records LLMYB_ETIMEOUT and every role unwinds.
#include <algorithm>

#include "paged.cuh"
#include "sm100.cuh"
#include "tma_host.h"

namespace llmyb {
namespace {

constexpr int kRows = 128;           // rows per tile = keys per block
constexpr int kBox = kRows * 128;    // 128 rows x 64 elements
constexpr int kThreads = 320;
constexpr uint32_t kTmemCols = 512;
constexpr int kJoinThreads = 256;

template <int D>
struct Layout {
  static constexpr int kTile = kRows * D * 2;
  static constexpr int kStages = D == 128 ? 5 : 8;  // K and V blocks alternate
  static constexpr int kQ = 0;                      // two query tiles
  static constexpr int kKV = 2 * kTile;
  static constexpr int kBar = kKV + kStages * kTile;
  static constexpr int kSmem = kBar + 256 + 1024;   // + alignment slack
};

struct PrefillArgs {
  PagedPool pool;
  const int32_t* cu_q;
  const int32_t* prefix;  // or null
  int32_t n_tokens, q_heads, group, tile_tokens, window, max_splits;
  float scale, softcap;
  const float* slopes;
  uint16_t* out;
  int64_t o_tok, o_head;
  float* lse;      // [n_tokens, q_heads] or null
  float* part_o;   // [splits][n_tokens][q_heads][D]
  float2* part_ml; // [splits][n_tokens][q_heads]
  int32_t* dev_status;
};

// Tokens of sequence b: the first one and how many.
__device__ __forceinline__ void tokens_of(const PrefillArgs& a, int b, int& q0, int& n) {
  q0 = max(0, min(a.cu_q[b], a.n_tokens));
  n = max(0, min(a.cu_q[b + 1], a.n_tokens) - q0);
}

// (sequence, two-tile piece) pairs of the batch and the splits of each key
// axis; by one warp.
__device__ __forceinline__ int plan(const PrefillArgs& a, int grid, int& splits) {
  const int lane = threadIdx.x & 31;
  int sum = 0;
  for (int b = lane; b < a.pool.batch; b += 32) {
    int q0, n;
    tokens_of(a, b, q0, n);
    sum += (n + 2 * a.tile_tokens - 1) / (2 * a.tile_tokens);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int units = sum * a.pool.kv_heads;
  splits = max(1, min(a.max_splits, units > 0 ? grid / units : 1));
  return units;
}

struct Unit {
  int b, q0, n, t0;    // sequence, its first token, its tokens, first token of the unit
  int kvh, split;
  int len, pos;        // length; position of token t0
  int lo, prefix;      // first key any row sees; prefix
  int kb0, blocks;     // key blocks [kb0, kb0 + blocks)
  int tiles;           // tiles with tokens: 1 or 2
};

// Unit u of the grid; by one warp.
__device__ __forceinline__ Unit unit_of(const PrefillArgs& a, int u, int splits) {
  const int lane = threadIdx.x & 31;
  const int per = a.pool.kv_heads * splits, step = 2 * a.tile_tokens;
  Unit x;
  x.b = 0;
  int before = 0, pieces = 0;
  for (int b0 = 0; b0 < a.pool.batch; b0 += 32) {
    int mine = 0;
    if (b0 + lane < a.pool.batch) {
      int q0, n;
      tokens_of(a, b0 + lane, q0, n);
      mine = (n + step - 1) / step;
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, (before + inc) * per > u);
    if (hit != 0) {
      const int l = __ffs(hit) - 1;
      x.b = b0 + l;
      pieces = __shfl_sync(0xffffffffu, mine, l);
      before += __shfl_sync(0xffffffffu, inc - mine, l);
      break;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  const int r = u - before * per;
  // the last tokens see the most keys: they start first
  const int piece = pieces - 1 - r / per;
  x.kvh = (r % per) / splits;
  x.split = r % splits;
  tokens_of(a, x.b, x.q0, x.n);
  x.t0 = piece * step;
  x.len = a.pool.length(x.b);
  x.pos = x.len - x.n + x.t0;
  const int count = min(step, x.n - x.t0);
  x.tiles = count > a.tile_tokens ? 2 : 1;
  x.prefix = a.prefix ? max(0, min(a.prefix[x.b], x.len)) : 0;
  const int last = x.pos + count - 1;
  int hi = last + 1;
  if (last >= 0) hi = max(hi, x.prefix);
  x.lo = a.window > 0 ? max(0, x.pos - a.window + 1) : 0;
  const int kb0 = x.lo / kRows, nblk = max(0, (hi + kRows - 1) / kRows - kb0);
  const int s0 = static_cast<int>(static_cast<int64_t>(nblk) * x.split / splits);
  const int s1 = static_cast<int>(static_cast<int64_t>(nblk) * (x.split + 1) / splits);
  x.kb0 = kb0 + s0;
  x.blocks = s1 - s0;
  return x;
}

// i-th unit of this CTA: heavy units come first in the list, and every other
// round runs backwards so that the rounds' differences cancel
__device__ __forceinline__ int unit_index(int i) {
  const int c = (i & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  return i * gridDim.x + c;
}

template <typename T>
constexpr uint32_t idesc(int n) {
  // D fp32; A and B bf16 (bits 7, 10) or fp16 (none)
  return sm100::make_idesc_bf16_f32(kRows, n) &
         (sizeof(T) == 2 && std::is_same<T, __half>::value ? ~((1u << 7) | (1u << 10)) : ~0u);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) paged_prefill_kernel(
    const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PrefillArgs a) {
  using L = Layout<D>;
  constexpr int kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* v_raw = bars + 2;       // values with rows to be zeroed
  uint64_t* mma_done = bars + 3;
  uint64_t* s_full = bars + 4;      // [2]
  uint64_t* p_full = bars + 6;      // [2]
  uint64_t* o_full = bars + 8;      // [2]
  uint64_t* kv_full = bars + 10;    // [kStages]
  uint64_t* kv_empty = kv_full + kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kv_empty + kStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) sm100::mbar_init(&bars[i], 1);
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(&s_full[i], 1);
      sm100::mbar_init(&p_full[i], 4);  // one arrival per softmax warp
      sm100::mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      sm100::mbar_init(&kv_full[i], 1);
      sm100::mbar_init(&kv_empty[i], 1);
    }
    *abort_flag = 0;
    sm100::fence_mbar_init();
    sm100::tma_prefetch_desc(&map_q);
    sm100::tma_prefetch_desc(&map_k);
    sm100::tma_prefetch_desc(&map_v);
  }
  if (warp == 9) sm100::tmem_alloc(tmem_slot, kTmemCols);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;
  int32_t* const status = a.dev_status;
  int splits;
  const int units = plan(a, gridDim.x, splits) * splits;

  if (warp == 8) {
    // ------------------------------------------------------------- TMA
    uint32_t n_kv = 0, n_q = 0, n_raw = 0;
    bool ok = true;
    const int page_rows = min(1 << a.pool.page_shift, kRows);  // rows per copy
    const int copies = kRows / page_rows * (D / 64);
    // the lane's copy of a block: page piece and 64-element half
    const int piece_row = lane / (D / 64) * page_rows, half = lane % (D / 64);
    for (int i = 0; ok; ++i) {
      const int u = unit_index(i);
      if (i * static_cast<int>(gridDim.x) >= units) break;
      if (u >= units) continue;
      const Unit x = unit_of(a, u, splits);
      if (x.blocks == 0) continue;
      if (!(ok = sm100::mbar_wait_warp(q_empty, (n_q & 1) ^ 1u, status, abort_flag))) break;
      if (lane == 0) {
        const uint32_t rows = a.tile_tokens * a.group;
        sm100::mbar_arrive_expect_tx(q_full, x.tiles * rows * D * 2);
        for (int t = 0; t < x.tiles; ++t)
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            sm100::tma_load_3d(&map_q, q_full, smem + L::kQ + t * L::kTile + c * kBox, c * 64,
                               x.kvh * a.group, x.q0 + x.t0 + t * a.tile_tokens);
      }
      ++n_q;
      const int32_t* row_table = a.pool.table + x.b * a.pool.table_stride;
      for (int j = x.blocks - 1; j >= 0 && ok; --j) {
        const int key0 = (x.kb0 + j) * kRows, key = key0 + piece_row;
        const bool held = lane < copies && key < x.len && key + page_rows > x.lo;
        int page = 0;
        if (held) {
          page = row_table[key >> a.pool.page_shift];
          if (page < 0 || page >= a.pool.num_pages) {
            report_status(status, LLMYB_EINVAL);
            page = 0;
          }
        }
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, held)) * page_rows * 128;
        const int in_page = key & ((1 << a.pool.page_shift) - 1);
        const bool mend = key0 + kRows > x.len || key0 < x.lo;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t s = n_kv % kStages, ph = (n_kv / kStages) & 1;
          if (!(ok = sm100::mbar_wait_warp(&kv_empty[s], ph ^ 1u, status, abort_flag))) break;
          uint8_t* dst = smem + L::kKV + s * L::kTile;
          uint64_t* bar = kv == 1 && mend ? v_raw : &kv_full[s];
          if (lane == 0) sm100::mbar_arrive_expect_tx(bar, bytes);
          __syncwarp();
          if (held)
            sm100::tma_load_4d(kv == 0 ? &map_k : &map_v, bar, dst + half * kBox + piece_row * 128,
                               half * 64, in_page, x.kvh, page);
          ++n_kv;
          if (kv == 1 && mend) {
            if (!(ok = sm100::mbar_wait_warp(v_raw, n_raw & 1, status, abort_flag))) break;
            ++n_raw;
            const int r0 = max(0, x.lo - key0), r1 = max(0, min(kRows, x.len - key0));
            for (int k = lane; k < kRows * 8 * (D / 64); k += 32) {
              const int r = (k >> 3) & (kRows - 1);
              if (r < r0 || r >= r1)
                *reinterpret_cast<uint4*>(dst + (k >> 10) * kBox + r * 128 + (k & 7) * 16) =
                    make_uint4(0, 0, 0, 0);
            }
            sm100::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&kv_full[s]);
          }
        }
      }
    }
    // no copy into shared memory may still be in flight at exit (after a
    // timeout; otherwise every one of these has been waited for)
    if (!ok) {
      if (n_q > 0) sm100::mbar_wait_warp(q_full, (n_q - 1) & 1, status, nullptr);
      for (uint32_t i = 1; i <= kStages && i <= n_kv; ++i)
        sm100::mbar_wait_warp(&kv_full[(n_kv - i) % kStages], ((n_kv - i) / kStages) & 1, status,
                              nullptr);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc_s = idesc<T>(kRows);
    constexpr uint32_t idesc_o = idesc<T>(D) | sm100::kIdescBMajorMN;
    const uint32_t q_addr = sm100::smem_u32(smem + L::kQ);
    const uint32_t kv_addr = sm100::smem_u32(smem + L::kKV);
    uint32_t n_kv = 0, n_q = 0, n_p[2] = {0, 0};
    bool ok = true;
    auto wait_kv = [&](uint32_t n) {
      return sm100::mbar_wait_warp(&kv_full[n % kStages], (n / kStages) & 1, status, abort_flag);
    };
    auto issue_s = [&](int t, uint32_t n) {  // S_t = Q_t K^T, K in load n
      if (lane == 0) {
        const uint32_t qa = q_addr + t * L::kTile, ka = kv_addr + (n % kStages) * L::kTile;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * kBox + (kk & 3) * 32;
          sm100::umma_bf16_ss(tmem + t * 128, sm100::make_sw128_kmajor_desc(qa + off),
                              sm100::make_sw128_kmajor_desc(ka + off), idesc_s, kk > 0 ? 1u : 0u);
        }
        sm100::umma_commit(&s_full[t]);
      }
      __syncwarp();
    };
    auto issue_pv = [&](int t, uint32_t n, bool first) {  // O_t (+)= P_t V, V in load n
      if (lane == 0) {
        const uint32_t va = kv_addr + (n % kStages) * L::kTile;
#pragma unroll
        for (int kk = 0; kk < kRows / 16; ++kk)
          sm100::umma_bf16_ts(tmem + 256 + t * D, tmem + t * 128 + kk * 8,
                              sm100::make_sw128_desc(va + kk * 2048, kBox, 1024), idesc_o,
                              (first && kk == 0) ? 0u : 1u);
      }
      __syncwarp();
    };
    auto commit = [&](uint64_t* bar) {
      if (lane == 0) sm100::umma_commit(bar);
      __syncwarp();
    };
    for (int i = 0; ok; ++i) {
      const int u = unit_index(i);
      if (i * static_cast<int>(gridDim.x) >= units) break;
      if (u >= units) continue;
      const Unit x = unit_of(a, u, splits);
      if (x.blocks == 0) continue;
      if (!(ok = sm100::mbar_wait_warp(q_full, n_q & 1, status, abort_flag) && wait_kv(n_kv)))
        break;
      ++n_q;
      sm100::tc_fence_after();
      for (int t = 0; t < x.tiles; ++t) issue_s(t, n_kv);
      commit(&kv_empty[n_kv % kStages]);
      if (x.blocks == 1) commit(q_empty);
      for (int j = 0; j < x.blocks && ok; ++j) {
        // load n_kv is the keys of block j, n_kv + 1 its values
        const bool more = j + 1 < x.blocks;
        if (!(ok = wait_kv(n_kv + 1))) break;
        for (int t = 0; t < x.tiles; ++t) {
          if (!(ok = sm100::mbar_wait_warp(&p_full[t], n_p[t] & 1, status, abort_flag))) break;
          ++n_p[t];
          sm100::tc_fence_after();
          issue_pv(t, n_kv + 1, j == 0);
          if (t == x.tiles - 1) commit(&kv_empty[(n_kv + 1) % kStages]);
          if (more) {
            if (t == 0 && !(ok = wait_kv(n_kv + 2))) break;
            issue_s(t, n_kv + 2);
            if (t == x.tiles - 1) {
              commit(&kv_empty[(n_kv + 2) % kStages]);
              if (j + 2 == x.blocks) commit(q_empty);
            }
          } else {
            commit(&o_full[t]);
          }
        }
        n_kv += 2;
      }
    }
    // every MMA completes before TMEM and shared memory go away
    commit(mma_done);
    sm100::mbar_wait_warp(mma_done, 0, status, nullptr);
  } else {
    // --------------------------------------------------------- softmax
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + t * 128, t_o = tmem + lanes + 256 + t * D;
    const int tok = row / a.group, g = row % a.group;  // token and head within the tile
    uint32_t n_s = 0, n_o = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      const int u = unit_index(i);
      if (i * static_cast<int>(gridDim.x) >= units) break;
      if (u >= units) continue;
      const Unit x = unit_of(a, u, splits);
      if (t >= x.tiles) continue;
      const int local = x.t0 + t * a.tile_tokens + tok;
      const bool live = tok < a.tile_tokens && local < x.n;
      const int head = x.kvh * a.group + g;
      const int pos = x.len - x.n + local;
      // visible keys of this row: lo <= j <= hi
      const int lo = a.window > 0 ? pos - a.window + 1 : 0;
      const int hi = pos < 0 ? -1 : max(pos, x.prefix - 1);
      // of every row of the tile: max lo, min hi
      const int first_pos = x.pos + t * a.tile_tokens;
      const int tile_hi = first_pos < 0 ? -1 : max(first_pos, x.prefix - 1);
      const int tile_lo = a.window > 0 ? first_pos + a.tile_tokens - a.window : 0;
      const float slope = a.slopes && live ? a.slopes[head] * kLog2e : 0.f;
      float m = -INFINITY, l = 0.f;
      for (int j = x.blocks - 1; j >= 0; --j) {
        if (!(ok = sm100::mbar_wait_warp(&s_full[t], n_s & 1, status, abort_flag))) break;
        ++n_s;
        sm100::tc_fence_after();
        uint32_t sr[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) sm100::tmem_ld_32x32b_x32(t_s + 32 * c, sr[c]);
        sm100::tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 4; ++c) sm100::tmem_regs_ready(sr[c]);
        const int j0 = (x.kb0 + j) * kRows;
        float sc = a.scale * kLog2e;
        if (a.softcap > 0.f) {
          const float in = a.scale / a.softcap, outer = a.softcap * kLog2e;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              sr[c][e] = __float_as_uint(outer * tanh_exp(__uint_as_float(sr[c][e]) * in));
          sc = 1.f;
        }
        if (a.slopes) {
          const float d0 = static_cast<float>(pos - j0);
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              sr[c][e] = __float_as_uint(fmaf(-slope, fabsf(d0 - (32 * c + e)),
                                              __uint_as_float(sr[c][e]) * sc));
          sc = 1.f;
        }
        if (j0 + kRows - 1 > tile_hi || j0 < tile_lo) {
          const int lo_c = lo - j0, hi_c = hi - j0;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * c + e < lo_c || 32 * c + e > hi_c) sr[c][e] = __float_as_uint(-INFINITY);
        }
        float mx[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) mx[e] = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e) mx[e & 7] = fmaxf(mx[e & 7], __uint_as_float(sr[c][e]));
        const float bm = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                               fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7]))) * sc;
        const bool raise = bm > m + 8.f;
        float alpha = 1.f;
        if (raise) {
          alpha = fast_exp2(m - bm);
          l *= alpha;
          m = bm;
        }
        if (__any_sync(0xffffffffu, raise) && j != x.blocks - 1) {
          // the scores of this block were issued behind the previous block's
          // product, so O is complete
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            sm100::tmem_ld_32x32b_x32(t_o + 32 * c, o);
            sm100::tmem_ld_wait();
            sm100::tmem_regs_ready(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            sm100::tmem_st_32x32b_x32(t_o + 32 * c, o);
          }
        }
        const float base = m == -INFINITY ? 0.f : -m;
        float rs[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float p0 = fast_exp2(fmaf(__uint_as_float(sr[c][2 * e]), sc, base));
            const float p1 = fast_exp2(fmaf(__uint_as_float(sr[c][2 * e + 1]), sc, base));
            rs[(2 * e) & 7] += p0;
            rs[(2 * e + 1) & 7] += p1;
            p[e] = Elem<T>::pack(p0, p1);
          }
          sm100::tmem_st_32x32b_x16(t_s + 16 * c, p);
        }
        l += ((rs[0] + rs[1]) + (rs[2] + rs[3])) + ((rs[4] + rs[5]) + (rs[6] + rs[7]));
        sm100::tmem_st_wait();
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      // ---------------------------------------------------- epilogue
      if (x.blocks > 0) {
        if (!(ok = sm100::mbar_wait_warp(&o_full[t], n_o & 1, status, abort_flag))) break;
        ++n_o;
        sm100::tc_fence_after();
      }
      const int64_t token = x.q0 + local;
      const int64_t at = (static_cast<int64_t>(x.split) * a.n_tokens + token) * a.q_heads + head;
      const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (x.blocks > 0) {
          sm100::tmem_ld_32x32b_x32(t_o + 32 * c, o);
          sm100::tmem_ld_wait();
          sm100::tmem_regs_ready(o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (!live) continue;
        if (splits > 1) {
          float4* dst = reinterpret_cast<float4*>(a.part_o + at * D + 32 * c);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                 __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
        } else {
          uint4* dst = reinterpret_cast<uint4*>(a.out + token * a.o_tok + head * a.o_head + 32 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = Elem<T>::pack(__uint_as_float(o[8 * e + 2 * k]) * inv,
                                   __uint_as_float(o[8 * e + 2 * k + 1]) * inv);
            dst[e] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (live) {
        if (splits > 1) a.part_ml[at] = make_float2(m, l);
        else if (a.lse) a.lse[token * a.q_heads + head] = lse_of(m, l);
      }
      sm100::tc_fence_before();  // O is read before the next unit's first product
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the splits: D / 4 threads per (token, head).
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) paged_prefill_join_kernel(PrefillArgs a, int grid) {
  constexpr int kVec = D / 4;
  int splits;
  plan(a, grid, splits);
  const int last = max(0, min(a.cu_q[a.pool.batch], a.n_tokens));
  const int first = max(0, min(a.cu_q[0], a.n_tokens));
  pdl_wait();
  if (splits <= 1) return;
  const int64_t rows = static_cast<int64_t>(a.n_tokens) * a.q_heads;
  const int64_t r = blockIdx.x * static_cast<int64_t>(kJoinThreads / kVec) + threadIdx.x / kVec;
  const int v = threadIdx.x % kVec;
  if (r >= static_cast<int64_t>(last) * a.q_heads || r < static_cast<int64_t>(first) * a.q_heads)
    return;
  float m = -INFINITY;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, a.part_ml[s * rows + r].x);
  const float base = m == -INFINITY ? 0.f : m;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float2 ml = a.part_ml[s * rows + r];
    const float4 x = *reinterpret_cast<const float4*>(a.part_o + (s * rows + r) * D + 4 * v);
    const float f = fast_exp2(ml.x - base);
    l = fmaf(ml.y, f, l);
    o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y);
    o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int64_t token = r / a.q_heads, head = r % a.q_heads;
  *reinterpret_cast<uint2*>(a.out + token * a.o_tok + head * a.o_head + 4 * v) =
      make_uint2(Elem<T>::pack(o.x * inv, o.y * inv), Elem<T>::pack(o.z * inv, o.w * inv));
  if (a.lse && v == 0) a.lse[r] = lse_of(m, l);
}

// 16-bit tensor of `rank` dimensions (innermost first, contiguous), boxes of
// 64 elements with the 128-byte swizzle; strides in elements.
bool make_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims,
              const int64_t* strides, const uint32_t* box) {
  auto enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  cuuint64_t d[5], st[4];
  cuuint32_t b[5], one[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = dims[i];
    b[i] = box[i];
    one[i] = 1;
    if (i > 0) st[i - 1] = static_cast<cuuint64_t>(strides[i]) * 2;
  }
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), d, st, b, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Splits of a key axis that can fill the GPU: every sequence has at most
// ceil(tokens / unit) units, so there are at least ceil(N / unit) of them.
int most_splits(int n_tokens, int kv_heads, int tile_tokens, int table_width, int page_size) {
  const int64_t units =
      ceil_div(n_tokens, 2 * tile_tokens) * static_cast<int64_t>(kv_heads);
  const int64_t blocks = ceil_div(static_cast<int64_t>(table_width) * page_size, kRows);
  return static_cast<int>(std::max<int64_t>(1, std::min(num_sms() / units, blocks)));
}

template <typename T, int D>
int32_t launch(const llmyb_paged_args* x, const PrefillArgs& a, cudaStream_t s) {
  using L = Layout<D>;
  int32_t st = ensure_smem(paged_prefill_kernel<T, D>, L::kSmem);
  if (st) return st;
  CUtensorMap mq, mk, mv;
  {
    const uint64_t dims[3] = {D, static_cast<uint64_t>(a.q_heads), static_cast<uint64_t>(a.n_tokens)};
    const int64_t strides[3] = {1, x->q_head_stride, x->q_token_stride};
    const uint32_t box[3] = {64, static_cast<uint32_t>(a.group), static_cast<uint32_t>(a.tile_tokens)};
    if (!make_map(&mq, x->q, 3, dims, strides, box)) return LLMYB_EUNSUPPORTED;
  }
  {
    const uint64_t dims[4] = {D, static_cast<uint64_t>(x->page_size),
                              static_cast<uint64_t>(a.pool.kv_heads),
                              static_cast<uint64_t>(a.pool.num_pages)};
    const int64_t strides[4] = {1, a.pool.row_stride, a.pool.head_stride, a.pool.page_stride};
    const uint32_t box[4] = {64, static_cast<uint32_t>(std::min(x->page_size, kRows)), 1, 1};
    if (!make_map(&mk, x->k_pages, 4, dims, strides, box) ||
        !make_map(&mv, x->v_pages, 4, dims, strides, box))
      return LLMYB_EUNSUPPORTED;
  }
  const int grid = num_sms();
  paged_prefill_kernel<T, D><<<grid, kThreads, L::kSmem, s>>>(mq, mk, mv, a);
  count_launch();
  st = launch_status();
  if (st || a.max_splits <= 1) return st;
  const int64_t ctas = ceil_div(static_cast<int64_t>(a.n_tokens) * a.q_heads, kJoinThreads / (D / 4));
  cudaError_t e = launch_pdl(paged_prefill_join_kernel<T, D>, dim3(static_cast<unsigned>(ctas)),
                             dim3(kJoinThreads), 0, s, a, grid);
  count_launch();
  return e == cudaSuccess ? launch_status() : static_cast<int32_t>(e);
}

}  // namespace
}  // namespace llmyb

using namespace llmyb;

LLMYB_API int64_t llmyb_paged_prefill_scratch_bytes(int32_t n_tokens, int32_t q_heads,
                                                    int32_t kv_heads, int32_t head_dim,
                                                    int32_t table_width, int32_t page_size) {
  if (n_tokens < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || head_dim <= 0 ||
      q_heads / kv_heads > kRows || table_width < 0 || page_size <= 0)
    return -1;
  if (n_tokens == 0) return 0;
  const int tile_tokens = kRows / (q_heads / kv_heads);
  const int64_t splits = most_splits(n_tokens, kv_heads, tile_tokens, table_width, page_size);
  if (splits <= 1) return 0;
  return splits * n_tokens * q_heads * (head_dim + 2) * 4;
}

LLMYB_API int32_t llmyb_paged_prefill(const llmyb_paged_args* x, void* stream) {
  int32_t st = paged_check(x);
  if (st) return st;
  st = paged_check_scores(x);
  if (st) return st;
  if (x->prefix && x->window > 0) return LLMYB_EINVAL;
  if (x->n_tokens == 0 || x->batch == 0) return LLMYB_OK;
  if (!x->cu_q) return LLMYB_EINVAL;
  const int group = x->q_heads / x->kv_heads;
  if (group > kRows || !paged_aligned(x->scratch)) return LLMYB_EUNSUPPORTED;
  PrefillArgs a;
  a.pool = paged_pool(x);
  a.cu_q = x->cu_q, a.prefix = x->prefix, a.n_tokens = x->n_tokens, a.q_heads = x->q_heads;
  a.group = group, a.tile_tokens = kRows / group;
  a.window = x->window, a.scale = x->scale, a.softcap = x->softcap, a.slopes = x->slopes;
  a.max_splits = most_splits(x->n_tokens, x->kv_heads, a.tile_tokens, x->table_width, x->page_size);
  if (a.max_splits > 1 && !x->scratch) return LLMYB_EINVAL;
  a.out = static_cast<uint16_t*>(x->out);
  a.o_tok = x->out_token_stride, a.o_head = x->out_head_stride;
  a.lse = x->lse;
  a.part_o = static_cast<float*>(x->scratch);
  a.part_ml = reinterpret_cast<float2*>(
      a.part_o + static_cast<int64_t>(a.max_splits) * x->n_tokens * x->q_heads * x->head_dim);
  a.dev_status = x->dev_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x->fp16) return x->head_dim == 64 ? launch<__half, 64>(x, a, s) : launch<__half, 128>(x, a, s);
  return x->head_dim == 64 ? launch<__nv_bfloat16, 64>(x, a, s)
                           : launch<__nv_bfloat16, 128>(x, a, s);
}
