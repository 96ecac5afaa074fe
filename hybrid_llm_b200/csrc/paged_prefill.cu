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
// tile wastes little on its diagonal.  A unit is two such tiles that run in
// turn over the same 128-key blocks, from the diagonal down:
//   warps 0-3, 4-7  softmax of tile 0 / 1 (one row per thread, TMEM lane = row)
//   warp 8          TMA: queries once per unit, keys and values page by page in
//                   one ring of 128-key blocks
//   warp 9          MMA: O_t += P_t V then S_t = Q_t K of the next block, for
//                   t = 0, 1: one tile's products run under the other's softmax
//   warp 10         checks the values of blocks that some row sees in part
// S in fp32 TMEM columns; P in 16 bits over S's first columns, the A operand of
// the second product; O in fp32 TMEM, divided by the weight sum at the end.
//
// The key blocks of all units form one list that is cut into equal ranges, one
// per CTA of a grid of one CTA per SM: prompts of any lengths load the SMs
// alike, and one chunk behind a long context uses all of them.  A unit that a
// range cuts leaves its unnormalised fp32 O, maxima and weight sums in scratch,
// and a second launch joins them in a fixed order.
//
// Values that a row does not see meet its zero weights, which do not cancel an
// infinity: in blocks that some row sees in part, rows outside the sequence
// (behind its end, or before the window; they may hold anything) are zeroed in
// shared memory, and so are values that are not finite, which are added to the
// outputs of the rows that see them (add_not_finite).  The check runs beside the
// block's softmax: 273 to 281 us for a ragged batch under a window, where about
// three of a unit's nine blocks are such edges.  All waits are bounded; a timeout
// records LLMYB_ETIMEOUT and every role unwinds.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "paged.cuh"
#include "sm100.cuh"
#include "tma_host.h"

namespace llmyb {
namespace {

constexpr int kRows = 128;         // rows per tile = keys per block
constexpr int kBox = kRows * 128;  // 128 rows x 64 elements
constexpr int kThreads = 384;
constexpr int kSoftmaxRegs = 192, kOtherRegs = 120;  // 256 x 192 + 128 x 120 = 384 x 168
constexpr uint32_t kTmemCols = 512;
constexpr int kJoinThreads = 256, kJoinRows = 32;
// What a unit costs beside its blocks (queries, first scores, the output), in blocks.
constexpr int kUnitCost = 3;
// Positions of a range at least, so that a range begins inside a unit or holds
// some of its blocks.
constexpr int kMinRange = 5;
// Up to this many blocks a unit is not cut: the second launch costs more.
constexpr int kWholeBlocks = 4;

template <int D>
struct Layout {
  static constexpr int kTile = kRows * D * 2;
  static constexpr int kStages = D == 128 ? 4 : 8;  // K and V blocks alternate
  static constexpr int kQ = 0;                      // two query tiles
  static constexpr int kKV = 2 * kTile;
  static constexpr int kOut = kKV + kStages * kTile;  // 4 KB per softmax warp
  static constexpr int kBar = kOut + 8 * 4096;
  static constexpr int kSmem = kBar + 512 + 1024;  // + alignment slack
};

// What a CTA leaves for the join: the cut unit that starts in its range, and
// whether its range begins inside one.
struct CutUnit {
  int32_t slot;            // -1: none starts here
  int32_t token, count;    // its first token and how many
  int32_t kvh;
  int32_t continues;       // the range begins inside a unit ...
  int32_t ends;            // ... and holds that unit's last block
};

struct PrefillArgs {
  PagedPool pool;
  const uint16_t* v_pages;  // for add_not_finite; the rest is read by TMA
  const int32_t* cu_q;
  const int32_t* prefix;  // or null
  int32_t n_tokens, q_heads, group, tile_tokens, window;
  int32_t cut;            // units may be cut
  float scale, softcap;
  const float* slopes;
  uint16_t* out;
  int64_t o_tok, o_head;
  float* lse;       // [n_tokens, q_heads] or null
  float* part_o;    // [grid * 2][D / 4][256][4]
  float2* part_ml;  // [grid * 2][256]
  CutUnit* cuts;    // [grid]
  int32_t* dev_status;
};

struct Seq {
  int q0, n, len, prefix;

  __device__ __forceinline__ void load(const PrefillArgs& a, int b) {
    q0 = max(0, min(a.cu_q[b], a.n_tokens));
    n = max(0, min(a.cu_q[b + 1], a.n_tokens) - q0);
    len = a.pool.length(b);
    prefix = a.prefix ? max(0, min(a.prefix[b], len)) : 0;
  }
  __device__ __forceinline__ int pieces(const PrefillArgs& a) const {
    return (n + 2 * a.tile_tokens - 1) / (2 * a.tile_tokens);
  }
};

// First key that the window leaves to a token at `pos`.  Positions go down to
// minus the token count (a length shorter than its tokens) and the window up to
// 2^31 - 1, so their difference is formed from position 0 on.
__device__ __forceinline__ int first_key(const PrefillArgs& a, int pos) {
  return a.window > 0 ? max(0, max(pos, 0) - a.window + 1) : 0;
}

// Key blocks [kb0, kb0 + count) that the tokens of one piece see.
__device__ __forceinline__ int piece_blocks(const PrefillArgs& a, const Seq& s, int piece, int& kb0,
                                            int& lo) {
  const int t0 = piece * 2 * a.tile_tokens, pos = s.len - s.n + t0;
  const int last = pos + min(2 * a.tile_tokens, s.n - t0) - 1;
  int hi = last + 1;
  if (last >= 0) hi = max(hi, s.prefix);
  lo = first_key(a, pos);
  kb0 = lo / kRows;
  return max(0, (hi + kRows - 1) / kRows - kb0);
}

// All pieces of the batch in order (sequence by sequence, last piece first),
// in chunks of 32: one lane per piece.  A group is the pieces of 32 sequences.
struct Group {
  int b0;     // first sequence
  Seq mine;   // of the lane's sequence
  int inc;    // pieces up to and with it
  int total;  // pieces of the group

  __device__ __forceinline__ void load(const PrefillArgs& a, int first) {
    const int lane = threadIdx.x & 31;
    b0 = first;
    mine = {0, 0, 0, 0};
    if (b0 + lane < a.pool.batch) mine.load(a, b0 + lane);
    inc = mine.pieces(a);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    total = __shfl_sync(0xffffffffu, inc, 31);
  }
  // Of the lane's piece in the chunk from p0: its weight (0: none), sequence
  // and number within it.
  __device__ __forceinline__ int weight(const PrefillArgs& a, int p0, int& b, int& piece) const {
    const int p = p0 + (threadIdx.x & 31);
    int l = 0;  // first lane whose running count exceeds p
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (__shfl_sync(0xffffffffu, inc, l + o - 1) <= p) l += o;
    const int end = __shfl_sync(0xffffffffu, inc, l);
    Seq s;
    s.q0 = 0;
    s.n = __shfl_sync(0xffffffffu, mine.n, l);
    s.len = __shfl_sync(0xffffffffu, mine.len, l);
    s.prefix = __shfl_sync(0xffffffffu, mine.prefix, l);
    b = b0 + l;
    piece = end - 1 - p;  // end - pieces <= p < end
    int kb0, lo;
    return p < total ? (piece_blocks(a, s, piece, kb0, lo) + kUnitCost) * a.pool.kv_heads : 0;
  }
};

// The range of one CTA and the unit that it begins in.
struct Start {
  int64_t begin, end;  // positions in the list of blocks and unit costs
  int64_t at;          // position of the first unit
  int b, piece, kvh;
};

// Chunk sums of a batch of more than one chunk; where it has more chunks than
// that (over 16,000 pieces), several share a sum.
constexpr int kSums = 512;

// numerator / denominator for values that mostly fit 32 bits
__device__ __forceinline__ int64_t divide(int64_t n, int64_t d) {
  if (((n | d) >> 32) == 0) return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
  return n / d;
}

// This CTA's range of `total` positions.
__device__ __forceinline__ void set_range(const PrefillArgs& a, int64_t total, Start& r) {
  // as many ranges as can have kMinRange positions (1 where units are not
  // cut); the CTAs behind have none
  const int64_t most = max(static_cast<int64_t>(1), a.cut ? divide(total, kMinRange) : total);
  const int64_t ranges = min(static_cast<int64_t>(gridDim.x), most);
  const int64_t c = min(static_cast<int64_t>(blockIdx.x), ranges);
  r.begin = divide(total * c, ranges);
  r.end = divide(total * min(c + 1, ranges), ranges);
}

// If position r.begin lies in this chunk (`before` positions come before it):
// the unit there.
__device__ __forceinline__ bool find_unit(const PrefillArgs& a, int w, int b, int piece,
                                          int64_t& before, Start& r) {
  const int lane = threadIdx.x & 31;
  int sum = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  const uint32_t hit = __ballot_sync(0xffffffffu, before + sum > r.begin);
  if (hit == 0) {
    before += __shfl_sync(0xffffffffu, sum, 31);
    return false;
  }
  const int h = __ffs(hit) - 1;
  r.b = __shfl_sync(0xffffffffu, b, h);
  r.piece = __shfl_sync(0xffffffffu, piece, h);
  const int unit = __shfl_sync(0xffffffffu, w, h) / a.pool.kv_heads;
  before += __shfl_sync(0xffffffffu, sum - w, h);
  r.kvh = static_cast<int>(r.begin - before) / unit;
  r.at = before + static_cast<int64_t>(r.kvh) * unit;
  return true;
}

// Before the roles part, by the whole CTA; the result is warp 0's.  Beyond one
// chunk every warp weighs some of them into shared memory (`sums`), and warp 0
// looks the range's first unit up.
__device__ __forceinline__ Start find_start(const PrefillArgs& a, int64_t* sums, int warps) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Start r = {0, 0, 0, a.pool.batch, 0, 0};
  Group g;
  g.load(a, 0);
  if (a.pool.batch <= 32 && g.total <= 32) {
    if (warp != 0) return r;
    int b, piece;
    const int w = g.weight(a, 0, b, piece);
    set_range(a, __reduce_add_sync(0xffffffffu, w), r);
    int64_t before = 0;
    if (r.begin < r.end) find_unit(a, w, b, piece, before, r);
    return r;
  }
  // chunks at most: one per 32 pieces and one per group; pieces at most: one
  // per unit's tokens and one per sequence
  const int64_t pieces = a.n_tokens / (2 * a.tile_tokens) + a.pool.batch;
  const int most = static_cast<int>(pieces / 32) + (a.pool.batch + 31) / 32 + 1;
  const int per = (most + kSums - 1) / kSums;
  for (int i = threadIdx.x; i < kSums; i += blockDim.x) sums[i] = 0;
  __syncthreads();
  int chunk = 0;
  for (int b0 = 0; b0 < a.pool.batch; b0 += 32) {
    if (b0 > 0) g.load(a, b0);
    for (int p0 = 0; p0 < g.total; p0 += 32, ++chunk) {
      if (chunk % warps != warp) continue;
      int b, piece;
      const int w = __reduce_add_sync(0xffffffffu, g.weight(a, p0, b, piece));
      if (lane == 0)
        atomicAdd(reinterpret_cast<unsigned long long*>(&sums[min(chunk / per, kSums - 1)]),
                  static_cast<unsigned long long>(w));
    }
  }
  __syncthreads();
  if (warp != 0) return r;
  int64_t mine = 0;  // of kSums / 32 neighbours
#pragma unroll
  for (int i = 0; i < kSums / 32; ++i) mine += sums[lane * (kSums / 32) + i];
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  set_range(a, __shfl_sync(0xffffffffu, inc, 31), r);
  if (r.begin >= r.end) return r;
  // the sum, then the chunk, then the piece that holds r.begin
  const int l = __ffs(__ballot_sync(0xffffffffu, inc > r.begin)) - 1;
  int64_t before = __shfl_sync(0xffffffffu, inc - mine, l);
  int at = l * (kSums / 32);
  while (before + sums[at] <= r.begin) before += sums[at++];
  chunk = 0;
  for (int b0 = 0; b0 < a.pool.batch; b0 += 32) {
    if (a.pool.batch > 32) g.load(a, b0);
    const int chunks = (g.total + 31) / 32;
    for (int k = max(0, at * per - chunk); k < chunks; ++k) {
      int b, piece;
      const int w = g.weight(a, 32 * k, b, piece);
      if (find_unit(a, w, b, piece, before, r)) return r;
    }
    chunk += chunks;
  }
  return r;
}

// A unit, or the part of it in one CTA's range, as the roles get it.
struct Unit {
  int blocks;         // key blocks [kb0, kb0 + blocks); -1: no more units
  int seq, len;       // sequence and its length
  int kb0, tiles;     // tiles with tokens
  int kvh;
  int token, count;   // first token, how many
  int pos;            // position of the first token
  int prefix;
  int starts, ends;   // the part holds the unit's last keys / first keys
  int first;          // first key that any row sees
  int lo, hi;         // the keys that every row sees
  int odd;            // values were left out for add_not_finite

  // some row does not see all keys of the block at j0
  __device__ __forceinline__ bool edge(int j0) const { return j0 + kRows - 1 > hi || j0 < lo; }
};

// The units of one CTA's range, in order.
struct Units {
  Start at;  // the next unit
  Seq s;
  int b, lo;  // sequence of the current unit; first key any of its rows sees

  __device__ __forceinline__ bool next(const PrefillArgs& a, Unit& u) {
    while (at.at < at.end && at.b < a.pool.batch) {
      if (at.piece < 0) {  // next sequence with tokens
        if (++at.b == a.pool.batch) break;
        s.load(a, at.b);
        at.piece = s.pieces(a) - 1;
        at.kvh = 0;
        continue;
      }
      int kb0;
      const int all = piece_blocks(a, s, at.piece, kb0, lo);
      const int64_t here = at.at;
      const int t0 = at.piece * 2 * a.tile_tokens;
      at.at += all + kUnitCost;
      b = at.b;
      u.kvh = at.kvh;
      if (++at.kvh == a.pool.kv_heads) {
        at.kvh = 0;
        --at.piece;
      }
      const bool first = here >= at.begin;  // the unit begins in this range
      int s0 = 0, s1 = all;                 // its blocks, counted from the last keys
      if (a.cut) {
        if (!first) s0 = min(all, max(0, static_cast<int>(at.begin - here) - kUnitCost));
        if (at.at > at.end) s1 = max(0, static_cast<int>(at.end - here) - kUnitCost);
      } else if (!first) {
        s1 = 0;
      }
      if (s0 >= s1 && !(all == 0 && first)) continue;
      u.blocks = s1 - s0;
      u.seq = b;
      u.kb0 = kb0 + all - s1;
      u.count = min(2 * a.tile_tokens, s.n - t0);
      u.tiles = u.count > a.tile_tokens ? 2 : 1;
      u.token = s.q0 + t0;
      u.pos = s.len - s.n + t0;
      u.prefix = s.prefix;
      u.len = s.len;
      u.first = lo;
      u.lo = first_key(a, u.pos + u.count - 1);
      u.hi = u.pos < 0 ? -1 : max(u.pos, u.prefix - 1);
      u.odd = 0;
      u.starts = s0 == 0;
      u.ends = s1 == all;
      return true;
    }
    return false;
  }
};

// A wait that polls: the suspending wait of sm100.cuh wakes up to a
// microsecond late, which the chain S -> P -> O pays twice per block
// (prefill of 8192 tokens: 769 us with it, 614 us polling).  Bounded like it.
// By a whole warp, whose lanes leave with one answer (what follows is for
// converged warps, after a timeout too): every lane polls for itself and one
// vote tells whether all have seen the phase complete.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int32_t* status,
                                     volatile int* abort_flag) {
  for (uint64_t t0 = 0;;) {
    bool ok = false;
    for (int i = 0; i < 4096 && !ok; ++i) ok = sm100::mbar_try_wait(bar, parity);
    if (__all_sync(0xffffffffu, ok)) return true;
    bool stop = abort_flag != nullptr && *abort_flag;
    const uint64_t now = globaltimer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > kWaitLimitNs) {
      report_status(status, LLMYB_ETIMEOUT);
      if (abort_flag != nullptr) *abort_flag = 1;
      stop = true;
    }
    if (__any_sync(0xffffffffu, stop)) return false;
  }
}

// elements e and e + 1 of a row of scores
__device__ __forceinline__ uint64_t pair(const uint32_t (&s)[128], int e) {
  return make2(__uint_as_float(s[e]), __uint_as_float(s[e + 1]));
}
__device__ __forceinline__ void set_pair(uint32_t (&s)[128], int e, uint64_t v) {
  const float2 x = split2(v);
  s[e] = __float_as_uint(x.x);
  s[e + 1] = __float_as_uint(x.y);
}

// Elements outside [lo, hi] become `other`: a word of 32 bits per 32 elements,
// whose bits go to predicates several at a time.
__device__ __forceinline__ void keep(uint32_t (&s)[128], int lo, int hi, uint32_t other) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    auto ones = [](int n) -> uint32_t { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; };
    const uint32_t in = ones(hi + 1 - 32 * c) & ~ones(lo - 32 * c);
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if ((in & (1u << e)) == 0) s[32 * c + e] = other;
  }
}

// largest of three, NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The bits of a packed pair's values that are not finite.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return ((w & e) == e ? 0xffffu : 0u) | ((w >> 16 & e) == e ? 0xffff0000u : 0u);
}

// Values that are not finite were left out of a unit's edge blocks, as rows see
// them that do not see their keys.  This adds them, from memory, to the stored
// outputs of the rows that do: with any weight they make an infinity or a NaN.  By
// a whole warp, a lane per row of the tile (dst, part: where its output is) and
// a lane per D / 32 columns; rare, and it reads the edge blocks' values alone.
template <typename T, int D>
__device__ __forceinline__ void add_not_finite(const PrefillArgs& a, const Unit& u, bool live, int lo,
                                               int hi, int64_t dst, float4* part) {
  constexpr int kWords = D / 64;  // column pairs of each lane
  const int lane = threadIdx.x & 31;
  const int32_t* const table = a.pool.table + u.seq * a.pool.table_stride;
  const int end = min((u.kb0 + u.blocks) * kRows, u.len);
  for (int k0 = max(u.kb0 * kRows, u.first & ~31); k0 < end; k0 += 32) {
    if (!u.edge(k0 & ~(kRows - 1))) continue;
    int64_t at = 0;  // a key per lane: its row within the pool
    if (k0 + lane < end) {
      const int key = k0 + lane;
      int page = table[key >> a.pool.page_shift];
      if (page < 0 || page >= a.pool.num_pages) page = 0;  // as the copies take it
      at = static_cast<int64_t>(page) * a.pool.page_stride + u.kvh * a.pool.head_stride +
           (key & ((1 << a.pool.page_shift) - 1)) * a.pool.row_stride;
    }
    const int count = min(32, end - k0);
    auto value = [&](int i, int c) -> uint32_t {  // bits that are not finite, of key k0 + i
      const uint16_t* const row = a.v_pages + __shfl_sync(0xffffffffu, at, i);
      const uint32_t w = *reinterpret_cast<const uint32_t*>(row + 2 * (kWords * lane + c));
      return w & not_finite<T>(w);
    };
    uint32_t keys = 0u;  // that have one
#pragma unroll 8
    for (int i = 0; i < count; ++i) {
      uint32_t any = 0u;
#pragma unroll
      for (int c = 0; c < kWords; ++c) any |= value(i, c);
      if (__any_sync(0xffffffffu, any != 0u)) keys |= 1u << i;
    }
    if (keys == 0u) continue;
    for (uint32_t rows = __ballot_sync(0xffffffffu, live); rows != 0u; rows &= rows - 1) {
      const int r = __ffs(rows) - 1;
      const int r_lo = __shfl_sync(0xffffffffu, lo, r) - k0, r_hi = __shfl_sync(0xffffffffu, hi, r) - k0;
      const int64_t r_dst = __shfl_sync(0xffffffffu, dst, r);
      float4* const r_part = reinterpret_cast<float4*>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(part), r));
      float2 sum[kWords] = {};
      for (uint32_t k = keys; k != 0u; k &= k - 1) {
        const int i = __ffs(k) - 1;
        if (i < r_lo || i > r_hi) continue;
#pragma unroll
        for (int c = 0; c < kWords; ++c) {
          const float2 x = Elem<T>::unpack(value(i, c));
          sum[c].x += x.x, sum[c].y += x.y;
        }
      }
#pragma unroll
      for (int c = 0; c < kWords; ++c) {
        if (sum[c].x == 0.f && sum[c].y == 0.f) continue;
        const int pair = kWords * lane + c;
        if (part != nullptr) {
          float2* const o = reinterpret_cast<float2*>(r_part + pair / 2 * 256) + pair % 2;
          *o = make_float2(o->x + sum[c].x, o->y + sum[c].y);
        } else {
          uint32_t* const o = reinterpret_cast<uint32_t*>(a.out + r_dst) + pair;
          const float2 x = Elem<T>::unpack(*o);
          *o = Elem<T>::pack(x.x + sum[c].x, x.y + sum[c].y);
        }
      }
    }
  }
}

template <typename T>
constexpr uint32_t idesc(int n) {
  // D fp32; A and B bf16 (bits 7, 10) or fp16 (none)
  return sm100::make_idesc_bf16_f32(kRows, n) &
         (std::is_same<T, __half>::value ? ~((1u << 7) | (1u << 10)) : ~0u);
}

template <typename T, int D, bool kCap, bool kBias>
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
  uint64_t* mma_done = bars + 2;
  uint64_t* s_full = bars + 3;      // [2]
  uint64_t* p_full = bars + 5;      // [2]
  uint64_t* o_full = bars + 7;      // [2]
  uint64_t* u_full = bars + 9;      // [2] units announced by the TMA warp
  uint64_t* u_empty = bars + 11;    // [2]
  uint64_t* kv_full = bars + 13;    // [kStages]
  uint64_t* kv_empty = kv_full + kStages;
  uint64_t* v_raw = kv_empty + kStages;  // [kStages] values of an edge block, unchecked
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_raw + kStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  Start* start = reinterpret_cast<Start*>(tmem_slot + 2);
  Unit* ring = reinterpret_cast<Unit*>(start + 1);  // [2]
  static_assert((13 + 3 * kStages) * 8 + 8 + sizeof(Start) + 2 * sizeof(Unit) <= 512, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 9) sm100::tmem_alloc(tmem_slot, kTmemCols);
  if (threadIdx.x == 352) {
    for (int i = 0; i < 3; ++i) sm100::mbar_init(&bars[i], 1);
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(&s_full[i], 1);
      sm100::mbar_init(&p_full[i], 4);  // one arrival per softmax warp
      sm100::mbar_init(&o_full[i], 1);
      sm100::mbar_init(&u_full[i], 1);
      sm100::mbar_init(&u_empty[i], 10);  // the softmax, MMA and checking warps
    }
    for (int i = 0; i < kStages; ++i) {
      sm100::mbar_init(&kv_full[i], 1);
      sm100::mbar_init(&kv_empty[i], 1);
      sm100::mbar_init(&v_raw[i], 1);
    }
    *abort_flag = 0;
    sm100::fence_mbar_init();
    sm100::tma_prefetch_desc(&map_q);
    sm100::tma_prefetch_desc(&map_k);
    sm100::tma_prefetch_desc(&map_v);
  }
  {
    // the sums lie where the first queries will: order them before the copies
    const Start r = find_start(a, reinterpret_cast<int64_t*>(smem + L::kQ), kThreads / 32);
    if (threadIdx.x == 0) *start = r;
    sm100::fence_proxy_async_smem();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;
  int32_t* const status = a.dev_status;
  if (a.cut && threadIdx.x == 0) a.cuts[blockIdx.x] = {-1, 0, 0, 0, 0, 0};
  // the next unit, for every role but TMA's (n: units so far); it stays in the
  // ring, out of the registers, until its role is done with it
  auto get = [&](uint32_t n) -> bool {
    return wait(&u_full[n & 1], (n >> 1) & 1, status, abort_flag) && ring[n & 1].blocks >= 0;
  };
  auto done = [&](uint32_t n) {
    __syncwarp();
    if (lane == 0) sm100::mbar_arrive(&u_empty[n & 1]);
  };

  // the register split is set inside the role branches: what follows a common
  // point would be compiled for the smaller share
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 8) {
      // ----------------------------------------------------------- TMA
      uint32_t n_kv = 0, n_q = 0;
      uint32_t raw = 0, raw_ph = 0;  // by stage: its last copy is an unchecked one; their phases
      bool ok = true;
      const int page_rows = min(1 << a.pool.page_shift, kRows);  // rows per copy
      const int copies = kRows / page_rows * (D / 64);
      // the lane's copy of a block: page piece and 64-element half
      const int piece_row = lane / (D / 64) * page_rows, half = lane % (D / 64);
      Units x;
      x.at = *start;
      if (x.at.b < a.pool.batch) x.s.load(a, x.at.b);
      for (uint32_t n = 0; ok; ++n) {
        Unit u;
        if (!x.next(a, u)) u.blocks = -1;
        if (!(ok = wait(&u_empty[n & 1], ((n >> 1) & 1) ^ 1u, status, abort_flag))) break;
        if (lane == 0) {
          ring[n & 1] = u;
          sm100::mbar_arrive(&u_full[n & 1]);
        }
        __syncwarp();
        if (u.blocks < 0) break;
        const int blocks = u.blocks, kb0 = u.kb0, len = x.s.len, lo = x.lo, kvh = u.kvh;
        if (blocks == 0) continue;
        if (!(ok = wait(q_empty, (n_q & 1) ^ 1u, status, abort_flag))) break;
        if (lane == 0) {
          sm100::mbar_arrive_expect_tx(q_full, u.tiles * a.tile_tokens * a.group * D * 2);
          for (int t = 0; t < u.tiles; ++t)
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              sm100::tma_load_3d(&map_q, q_full, smem + L::kQ + t * L::kTile + c * kBox, c * 64,
                                 kvh * a.group, u.token + t * a.tile_tokens);
        }
        ++n_q;
        const int32_t* row_table = a.pool.table + x.b * a.pool.table_stride;
        for (int j = blocks - 1; j >= 0 && ok; --j) {
          const int key0 = (kb0 + j) * kRows, key = key0 + piece_row;
          const bool held = lane < copies && key < len && key + page_rows > lo;
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
          const bool edge = u.edge(key0);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const uint32_t s = n_kv % kStages, ph = (n_kv / kStages) & 1;
            if (!(ok = wait(&kv_empty[s], ph ^ 1u, status, abort_flag))) break;
            uint8_t* dst = smem + L::kKV + s * L::kTile;
            const bool check = kv == 1 && edge;
            uint64_t* bar = check ? &v_raw[s] : &kv_full[s];
            raw = (raw & ~(1u << s)) | (check ? 1u << s : 0u);
            if (check) raw_ph ^= 1u << s;
            if (lane == 0) sm100::mbar_arrive_expect_tx(bar, bytes);
            __syncwarp();
            if (held)
              sm100::tma_load_4d(kv == 0 ? &map_k : &map_v, bar, dst + half * kBox + piece_row * 128,
                                 half * 64, in_page, kvh, page);
            ++n_kv;
          }
        }
      }
      // no copy into shared memory may still be in flight at exit (after a
      // timeout; otherwise every one of these has been waited for)
      if (!ok) {
        if (n_q > 0) wait(q_full, (n_q - 1) & 1, status, nullptr);
        for (uint32_t i = 1; i <= kStages && i <= n_kv; ++i) {
          const uint32_t n = n_kv - i, s = n % kStages;
          if (raw >> s & 1) wait(&v_raw[s], (raw_ph >> s & 1) ^ 1u, status, nullptr);
          else wait(&kv_full[s], (n / kStages) & 1, status, nullptr);
        }
      }
    } else if (warp == 9) {
      // ---------------------------------------------------- MMA issuer
      constexpr uint32_t idesc_s = idesc<T>(kRows);
      constexpr uint32_t idesc_o = idesc<T>(D) | sm100::kIdescBMajorMN;
      // This warp shares its scheduler with softmax warps and issues a product
      // every 64 cycles, so its instructions count: one elected thread issues
      // (with lane == 0 in its place the operands went through per-thread
      // registers: 609 us against 558), and descriptors are made once, tiles
      // and steps differing in the address field alone (538 us against 484;
      // shared memory ends below 2^18, so the field does not overflow).
      const uint64_t q_desc = sm100::make_sw128_kmajor_desc(sm100::smem_u32(smem + L::kQ));
      const uint64_t k_desc = sm100::make_sw128_kmajor_desc(sm100::smem_u32(smem + L::kKV));
      const uint64_t v_desc = sm100::make_sw128_desc(sm100::smem_u32(smem + L::kKV), kBox, 1024);
      uint32_t n_kv = 0, n_q = 0, n_p[2] = {0, 0};
      bool ok = true;
      auto wait_kv = [&](uint32_t n) {
        return wait(&kv_full[n % kStages], (n / kStages) & 1, status, abort_flag);
      };
      auto issue_s = [&](int t, uint32_t n) {  // S_t = Q_t K^T, K in load n
        if (sm100::elect_one()) {
          const uint64_t qd = q_desc + t * (L::kTile >> 4);
          const uint64_t kd = k_desc + (n % kStages) * (L::kTile >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * kBox + (kk & 3) * 32) >> 4;
            sm100::umma_bf16_ss(tmem + t * 128, qd + off, kd + off, idesc_s, kk > 0 ? 1u : 0u);
          }
          sm100::umma_commit(&s_full[t]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int t, uint32_t n, bool first) {  // O_t (+)= P_t V, V in load n
        if (sm100::elect_one()) {
          const uint64_t vd = v_desc + (n % kStages) * (L::kTile >> 4);
#pragma unroll
          for (int kk = 0; kk < kRows / 16; ++kk)
            sm100::umma_bf16_ts(tmem + 256 + t * D, tmem + t * 128 + kk * 8,
                                vd + kk * (2048 >> 4), idesc_o, (first && kk == 0) ? 0u : 1u);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (sm100::elect_one()) sm100::umma_commit(bar);
        __syncwarp();
      };
      for (uint32_t n = 0; ok && get(n); ++n) {
        const int blocks = ring[n & 1].blocks, tiles = ring[n & 1].tiles;
        done(n);
        if (blocks == 0) continue;
        if (!(ok = wait(q_full, n_q & 1, status, abort_flag) && wait_kv(n_kv))) break;
        ++n_q;
        sm100::tc_fence_after();
        for (int t = 0; t < tiles; ++t) issue_s(t, n_kv);
        commit(&kv_empty[n_kv % kStages]);
        if (blocks == 1) commit(q_empty);
        for (int j = 0; j < blocks && ok; ++j) {
          // load n_kv is the keys of block j, n_kv + 1 its values
          const bool more = j + 1 < blocks;
          if (!(ok = wait_kv(n_kv + 1))) break;
          for (int t = 0; t < tiles; ++t) {
            if (!(ok = wait(&p_full[t], n_p[t] & 1, status, abort_flag))) break;
            ++n_p[t];
            sm100::tc_fence_after();
            issue_pv(t, n_kv + 1, j == 0);
            if (t == tiles - 1) commit(&kv_empty[(n_kv + 1) % kStages]);
            if (more) {
              if (t == 0 && !(ok = wait_kv(n_kv + 2))) break;
              issue_s(t, n_kv + 2);
              if (t == tiles - 1) {
                commit(&kv_empty[(n_kv + 2) % kStages]);
                if (j + 2 == blocks) commit(q_empty);
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
      wait(mma_done, 0, status, nullptr);
    } else if (warp == 10) {
      // ------------------------------------------- values of edge blocks
      // A block that some row sees in part: zero weights meet its other values.
      // Rows outside the sequence are zeroed, they may hold anything; values
      // that are not finite are zeroed and added by the softmax warps to the rows
      // that see them.  Beside the block's first product and softmax, which
      // take longer.
      uint32_t n_kv = 0, ph = 0;  // ph: phases of v_raw
      bool ok = true;
      for (uint32_t n = 0; ok && get(n); ++n) {
        const Unit& u = ring[n & 1];
        for (int j = u.blocks - 1; j >= 0; --j, n_kv += 2) {
          const int key0 = (u.kb0 + j) * kRows;
          if (!u.edge(key0)) continue;
          const uint32_t s = (n_kv + 1) % kStages;
          if (!(ok = wait(&v_raw[s], ph >> s & 1, status, abort_flag))) break;
          ph ^= 1u << s;
          uint4* const v = reinterpret_cast<uint4*>(smem + L::kKV + s * L::kTile);
          const int r0 = max(0, u.first - key0), r1 = max(0, min(kRows, u.len - key0));
          constexpr int kPieces = kRows * 8 * (D / 64);  // of 16 bytes, eight a row and box
          if (r0 > 0 || r1 < kRows) {
            for (int k = lane; k < kPieces; k += 32) {
              const int r = k >> 3 & (kRows - 1);
              if (r < r0 || r >= r1) v[k] = make_uint4(0, 0, 0, 0);
            }
            __syncwarp();
          }
          uint32_t acc[4] = {0u, 0u, 0u, 0u};
#pragma unroll 1
          for (int k = lane; k < kPieces; k += 32 * 8) {
            uint4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = v[k + 32 * i];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              acc[0] = Elem<T>::probe(x[i].x, acc[0]), acc[1] = Elem<T>::probe(x[i].y, acc[1]);
              acc[2] = Elem<T>::probe(x[i].z, acc[2]), acc[3] = Elem<T>::probe(x[i].w, acc[3]);
            }
          }
          const uint32_t found = not_finite<T>(acc[0]) | not_finite<T>(acc[1]) |
                                 not_finite<T>(acc[2]) | not_finite<T>(acc[3]);
          if (__builtin_expect(__any_sync(0xffffffffu, found), 0)) {
            for (int k = lane; k < kPieces; k += 32) {
              const uint4 x = v[k];
              v[k] = make_uint4(x.x & ~not_finite<T>(x.x), x.y & ~not_finite<T>(x.y),
                                x.z & ~not_finite<T>(x.z), x.w & ~not_finite<T>(x.w));
            }
            if (lane == 0) ring[n & 1].odd = 1;  // before the arrival
          }
          sm100::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) sm100::mbar_arrive(&kv_full[s]);
        }
        done(n);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // --------------------------------------------------------- softmax
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + t * 128, t_o = tmem + lanes + 256 + t * D;
    const int tok = row / a.group, g = row % a.group;  // token and head within the tile
    uint32_t n_s = 0, n_o = 0;
    bool ok = true;
    for (uint32_t n = 0; ok && get(n); ++n) {
      const Unit& u = ring[n & 1];
      if (threadIdx.x == 0 && !(u.starts && u.ends)) {
        CutUnit& cut = a.cuts[blockIdx.x];
        if (u.starts) {
          cut.slot = 1, cut.token = u.token, cut.count = u.count, cut.kvh = u.kvh;
        } else {
          cut.continues = 1, cut.ends = u.ends;
        }
      }
      if (t >= u.tiles) {
        done(n);
        continue;
      }
      float m = -INFINITY, l = 0.f;  // l: this row's weights by 2^-m
      const int blocks = u.blocks;
      const int local = t * a.tile_tokens + tok;  // within the unit
      const bool live = tok < a.tile_tokens && local < u.count;
      const int pos = u.pos + local;
      // visible keys of this row: lo <= j <= hi
      const int lo = first_key(a, pos);
      const int hi = pos < 0 ? -1 : max(pos, u.prefix - 1);
      // of every row of the tile: max lo, min hi
      const int first_pos = u.pos + t * a.tile_tokens;
      const int tile_hi = first_pos < 0 ? -1 : max(first_pos, u.prefix - 1);
      const int tile_lo = first_key(a, first_pos + a.tile_tokens - 1);
      const float slope = kBias && live ? a.slopes[u.kvh * a.group + g] * kLog2e : 0.f;
      bool settled = false;  // every live row of the warp has its first maximum
      const int kb0 = u.kb0;
      const bool ahead = kBias && u.prefix != 0;
      for (int j = blocks - 1; j >= 0; --j) {
        if (!(ok = wait(&s_full[t], n_s & 1, status, abort_flag))) break;
        ++n_s;
        sm100::tc_fence_after();
        uint32_t sr[128];
        {
          uint32_t part[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) sm100::tmem_ld_32x32b_x32(t_s + 32 * c, part[c]);
          sm100::tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 4; ++c) sm100::tmem_regs_ready(part[c]);
#pragma unroll
          for (int e = 0; e < 128; ++e) sr[e] = part[e / 32][e % 32];
        }
        const int j0 = (kb0 + j) * kRows;
        float sc = a.scale * kLog2e;
        const bool edge = j0 + kRows - 1 > tile_hi || j0 < tile_lo;
        const int lo_c = lo - j0, hi_c = hi - j0;
        if constexpr (kCap) {
          if (__builtin_expect(edge, 0)) {  // what is not visible chooses no path below
            keep(sr, lo_c, hi_c, 0u);
          }
          // cap tanh(s / cap): the short form where every row of the warp has
          // |s| < cap, which one bit of 2 s / cap tells; the long one gives such
          // scores the same result
          const float in = 2.f * a.scale / a.softcap;
          const uint64_t in2 = make2(in, in);
          uint32_t big = 0u;
#pragma unroll
          for (int e = 0; e < 128; e += 2) {
            set_pair(sr, e, mul2(pair(sr, e), in2));
            big |= sr[e] | sr[e + 1];
          }
          const bool wide = live && (big & 0x40000000u);
          if (__builtin_expect(__any_sync(0xffffffffu, wide), 0)) {
#pragma unroll
            for (int e = 0; e < 128; e += 2) set_pair(sr, e, tanh_half2(pair(sr, e)));
          } else {
#pragma unroll
            for (int e = 0; e < 128; e += 2) set_pair(sr, e, tanh_half_poly2(pair(sr, e)));
          }
          sc = a.softcap * kLog2e;
        }
        if constexpr (kBias) {
          const float d0 = static_cast<float>(pos - j0);
          if (!ahead || j0 + kRows - 1 <= first_pos) {  // no visible key is ahead
            const uint64_t step = make2(slope, slope), sc2 = make2(sc, sc);
            const uint64_t b0 = make2(-slope * d0, -slope * d0);
#pragma unroll
            for (int e = 0; e < 128; e += 2)
              set_pair(sr, e,
                       fma2(pair(sr, e), sc2,
                            fma2(step, make2(static_cast<float>(e), static_cast<float>(e + 1)), b0)));
          } else {
#pragma unroll
            for (int e = 0; e < 128; ++e)
              sr[e] = __float_as_uint(fmaf(-slope, fabsf(d0 - e), __uint_as_float(sr[e]) * sc));
          }
          sc = 1.f;
        }
        if (__builtin_expect(edge, 0)) keep(sr, lo_c, hi_c, 0xff800000u);  // -inf
        // m of the rows that ask for it (and of no other: a row's result does not
        // depend on its neighbours) to the block's maximum (less kPrefillUp), l and
        // O rescaled
        auto raise = [&](bool ask) {
          float mx[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = __uint_as_float(sr[e]);
#pragma unroll
          for (int e = 4; e < 124; e += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mx[k] = max3(mx[k], __uint_as_float(sr[e + 2 * k]), __uint_as_float(sr[e + 2 * k + 1]));
          mx[0] = max3(mx[0], __uint_as_float(sr[124]), __uint_as_float(sr[125]));
          mx[1] = max3(mx[1], __uint_as_float(sr[126]), __uint_as_float(sr[127]));
          const float bm =
              fmaf(max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]), sc, -Elem<T>::kPrefillUp);
          float alpha = 1.f;
          if (ask && bm > m) {
            alpha = fast_exp2(m - bm);
            m = bm;
            l *= alpha;
          }
          if (j != blocks - 1) {
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
        };
        // P = 2^(s - m) to TMEM in the cache's type, the operand that the tensor
        // cores take (each off by at most half a step, unbiased: errors against 64
        // bits 0.0018-0.0024 of the output's size, its own rounding 0.0015-0.0017),
        // and its row sum, unrounded
        auto weights = [&]() -> float {
          const float base = m == -INFINITY ? 0.f : -m;
          const uint64_t sc2 = make2(sc, sc), base2 = make2(base, base);
          uint64_t rs[2] = {0ull, 0ull};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t p[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float2 w = split2(fma2(pair(sr, 32 * c + 2 * e), sc2, base2));
              w.x = fast_exp2(w.x), w.y = fast_exp2(w.y);
              rs[e & 1] = add2(rs[e & 1], make2(w.x, w.y));
              p[e] = Elem<T>::pack(w.x, w.y);
            }
            sm100::tmem_st_32x32b_x16(t_s + 16 * c, p);
          }
          const float2 r = split2(add2(rs[0], rs[1]));
          return r.x + r.y;
        };
        // The weights take the maximum of the blocks before.  Their sum shows
        // whether that is still near enough: below kMostWeight every one is
        // (fp16 holds 65504, sums are fp32), and the block's own maximum is never
        // formed (459 us against 502 with it).  Else, a NaN among them
        // included, and at a row's first keys it is.
        if (!settled) {
          const bool fresh = live && m == -INFINITY && hi >= j0;
          if (__any_sync(0xffffffffu, fresh)) raise(fresh);
          settled = __all_sync(0xffffffffu, !live || m != -INFINITY);
        }
        float sum = weights();
        const bool far = live && !(sum <= Elem<T>::kMostWeight);
        if (__builtin_expect(__any_sync(0xffffffffu, far), 0)) {
          raise(far);
          sum = weights();
        }
        l += sum;
        sm100::tmem_st_wait();
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      // ---------------------------------------------------- epilogue
      if (blocks > 0) {
        if (!(ok = wait(&o_full[t], n_o & 1, status, abort_flag))) break;
        ++n_o;
        sm100::tc_fence_after();
      }
      const float inv = inv_of(l);
      const bool whole = u.starts && u.ends;
      const int head = u.kvh * a.group + g;
      // This row's place in the output; the rows go there by way of shared
      // memory, 64 columns at a time, so that a store instruction writes whole
      // 128-byte lines (one row per thread: four times as long).
      const int64_t dst = live ? static_cast<int64_t>(u.token + local) * a.o_tok + head * a.o_head : -1;
      uint8_t* const stage = smem + L::kOut + warp * 4096;
      float4* const part = reinterpret_cast<float4*>(a.part_o) +
                           (2ll * blockIdx.x + (u.starts ? 1 : 0)) * (256 * D / 4) + t * kRows + row;
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {
        uint32_t o[2][32];
#pragma unroll
        for (int h = 0; h < 2; ++h) sm100::tmem_ld_32x32b_x32(t_o + 64 * c + 32 * h, o[h]);
        sm100::tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < 2; ++h) sm100::tmem_regs_ready(o[h]);
        if (blocks == 0) {
#pragma unroll
          for (int e = 0; e < 64; ++e) o[e / 32][e % 32] = 0u;
        }
        if (!whole) {  // column quads by row: the lanes' 16 bytes are neighbours
#pragma unroll
          for (int e = 0; e < 16; ++e)
            part[(16 * c + e) * 256] = make_float4(
                __uint_as_float(o[e / 8][4 * (e % 8)]), __uint_as_float(o[e / 8][4 * (e % 8) + 1]),
                __uint_as_float(o[e / 8][4 * (e % 8) + 2]), __uint_as_float(o[e / 8][4 * (e % 8) + 3]));
          continue;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = Elem<T>::pack(__uint_as_float(o[e / 4][8 * (e % 4) + 2 * k]) * inv,
                                 __uint_as_float(o[e / 4][8 * (e % 4) + 2 * k + 1]) * inv);
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((e ^ (lane & 7)) << 4)) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        uint4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r = 4 * k + (lane >> 3);
          v[k] = *reinterpret_cast<const uint4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int64_t at = __shfl_sync(0xffffffffu, dst, 4 * k + (lane >> 3));
          if (at >= 0) *reinterpret_cast<uint4*>(a.out + at + 64 * c + 8 * (lane & 7)) = v[k];
        }
        __syncwarp();
      }
      if (live) {
        if (!whole)
          a.part_ml[(2ll * blockIdx.x + (u.starts ? 1 : 0)) * 256 + t * kRows + row] = make_float2(m, l);
        else if (a.lse)
          a.lse[static_cast<int64_t>(u.token + local) * a.q_heads + head] = lse_of(m, l);
      }
      if (__builtin_expect(u.odd, 0)) {
        __syncwarp();  // behind the rows' stores
        add_not_finite<T, D>(a, u, live, lo, hi, dst, whole ? nullptr : part);
      }
      sm100::tc_fence_before();  // O is read before the next unit's first product
      done(n);
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the cut units: CTA (c, y) takes 32 rows of the one that starts in
// range c; its other pieces are the first ones of the ranges behind.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) paged_prefill_join_kernel(PrefillArgs a, int grid) {
  constexpr int kWarps = kJoinThreads / 32;
  __shared__ uint2 s_out[32][D / 4 + 1];
  pdl_wait();
  const CutUnit u = a.cuts[blockIdx.x];
  if (u.slot < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // its pieces lie in ranges [blockIdx.x, end)
  int end = blockIdx.x + 1;
  for (bool more = true; more; ) {
    const int c = end + lane;
    CutUnit n = {0, 0, 0, 0, 0, 0};
    if (c < grid) n = a.cuts[c];
    const uint32_t stop = __ballot_sync(0xffffffffu, !n.continues || n.ends);
    const int last = __ffs(stop) - 1;  // -1: all 32 go on
    more = stop == 0;
    end += more ? 32 : last + (__shfl_sync(0xffffffffu, n.continues, max(last, 0)) ? 1 : 0);
  }
  const int row0 = blockIdx.y * kJoinRows, r = row0 + lane;
  const int tok = r / kRows * a.tile_tokens + r % kRows / a.group;
  const bool live = r % kRows / a.group < a.tile_tokens && tok < u.count;
  auto slot = [&](int c) -> int64_t { return 2ll * c + (c == blockIdx.x ? 1 : 0); };
  float m = -INFINITY, l = 0.f;
  if (live) {
#pragma unroll 4
    for (int c = blockIdx.x; c < end; ++c) m = fmaxf(m, a.part_ml[slot(c) * 256 + r].x);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (int c = blockIdx.x; c < end; ++c) {
      const float2 ml = a.part_ml[slot(c) * 256 + r];
      l = fmaf(ml.y, fast_exp2(ml.x - base), l);
    }
    const float inv = inv_of(l);
    constexpr int kQuads = D / 4 / kWarps;  // column quads of this thread
    float4 o[kQuads];
#pragma unroll
    for (int k = 0; k < kQuads; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int c = blockIdx.x; c < end; ++c) {
      const float f = fast_exp2(a.part_ml[slot(c) * 256 + r].x - base);
      const float4* const from =
          reinterpret_cast<const float4*>(a.part_o) + (slot(c) * (D / 4) + warp) * 256 + r;
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        const float4 x = from[k * kWarps * 256];
        o[k].x = fmaf(x.x, f, o[k].x), o[k].y = fmaf(x.y, f, o[k].y);
        o[k].z = fmaf(x.z, f, o[k].z), o[k].w = fmaf(x.w, f, o[k].w);
      }
    }
#pragma unroll
    for (int k = 0; k < kQuads; ++k)
      s_out[lane][warp + k * kWarps] = make_uint2(Elem<T>::pack(o[k].x * inv, o[k].y * inv),
                                                  Elem<T>::pack(o[k].z * inv, o[k].w * inv));
    if (warp == 0 && a.lse)
      a.lse[static_cast<int64_t>(u.token + tok) * a.q_heads + u.kvh * a.group + r % kRows % a.group] =
          lse_of(m, l);
  }
  __syncthreads();
  for (int i = warp; i < kJoinRows; i += kWarps) {
    const int q = row0 + i, t = q / kRows * a.tile_tokens + q % kRows / a.group;
    if (q % kRows / a.group >= a.tile_tokens || t >= u.count) continue;
    uint16_t* dst = a.out + static_cast<int64_t>(u.token + t) * a.o_tok +
                    (u.kvh * a.group + q % kRows % a.group) * a.o_head;
    if (lane < D / 4) reinterpret_cast<uint2*>(dst)[lane] = s_out[i][lane];
  }
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

// Whether units may be cut: not where a sequence has few key blocks.
bool may_cut(int table_width, int page_size) {
  return ceil_div(static_cast<int64_t>(table_width) * page_size, kRows) > kWholeBlocks;
}

template <typename T, int D, bool kCap, bool kBias>
int32_t launch(const llmyb_paged_args* x, const PrefillArgs& a, cudaStream_t s) {
  using L = Layout<D>;
  auto* const kernel = paged_prefill_kernel<T, D, kCap, kBias>;
  int32_t st = ensure_smem(kernel, L::kSmem);
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
  kernel<<<grid, kThreads, L::kSmem, s>>>(mq, mk, mv, a);
  count_launch();
  st = launch_status();
  if (st || !a.cut) return st;
  const cudaError_t e = launch_pdl(paged_prefill_join_kernel<T, D>, dim3(grid, 256 / kJoinRows),
                                   dim3(kJoinThreads), 0, s, a, grid);
  count_launch();
  return e == cudaSuccess ? launch_status() : static_cast<int32_t>(e);
}

// The score transforms are compiled in or out: their code between the loads
// and the exponentials costs every block instruction fetches.
template <typename T, int D>
int32_t launch(const llmyb_paged_args* x, const PrefillArgs& a, cudaStream_t s) {
  if (a.softcap > 0.f)
    return a.slopes ? launch<T, D, true, true>(x, a, s) : launch<T, D, true, false>(x, a, s);
  return a.slopes ? launch<T, D, false, true>(x, a, s) : launch<T, D, false, false>(x, a, s);
}

}  // namespace
}  // namespace llmyb

using namespace llmyb;

LLMYB_API int64_t llmyb_paged_prefill_scratch_bytes(int32_t q_heads, int32_t kv_heads,
                                                    int32_t head_dim, int32_t table_width,
                                                    int32_t page_size) {
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || head_dim <= 0 ||
      q_heads / kv_heads > kRows || table_width < 0 || page_size <= 0)
    return -1;
  if (!may_cut(table_width, page_size)) return 0;
  return static_cast<int64_t>(num_sms()) * (2 * 256 * (head_dim + 2) * 4 + sizeof(CutUnit));
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
  // the weights of 32 pieces are added in 32 bits
  const int64_t blocks = ceil_div(static_cast<int64_t>(x->table_width) * x->page_size, kRows);
  if ((blocks + kUnitCost) * x->kv_heads >= 1ll << 26) return LLMYB_EUNSUPPORTED;
  PrefillArgs a;
  a.pool = paged_pool(x);
  a.v_pages = static_cast<const uint16_t*>(x->v_pages);
  a.cu_q = x->cu_q, a.prefix = x->prefix, a.n_tokens = x->n_tokens, a.q_heads = x->q_heads;
  a.group = group, a.tile_tokens = kRows / group;
  a.window = x->window, a.scale = x->scale, a.softcap = x->softcap, a.slopes = x->slopes;
  a.cut = may_cut(x->table_width, x->page_size);
  if (a.cut && !x->scratch) return LLMYB_EINVAL;
  a.out = static_cast<uint16_t*>(x->out);
  a.o_tok = x->out_token_stride, a.o_head = x->out_head_stride;
  a.lse = x->lse;
  const int64_t slots = 2ll * num_sms();
  a.part_o = static_cast<float*>(x->scratch);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + slots * 256 * x->head_dim);
  a.cuts = reinterpret_cast<CutUnit*>(a.part_ml + slots * 256);
  a.dev_status = x->dev_status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x->fp16) return x->head_dim == 64 ? launch<__half, 64>(x, a, s) : launch<__half, 128>(x, a, s);
  return x->head_dim == 64 ? launch<__nv_bfloat16, 64>(x, a, s)
                           : launch<__nv_bfloat16, 128>(x, a, s);
}
