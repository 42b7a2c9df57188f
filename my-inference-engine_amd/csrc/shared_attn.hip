// Attention of packed new tokens over a paged cache, keys that rows share read once.
//
// The softmax of a query over its keys is the merge of softmaxes over disjoint ranges of them: with
// m = max s, l = sum e^(s - m), O = sum e^(s - m) v of each range, M = max m:
//   L = sum l e^(m - M), O = sum O e^(m - M) / L.
// So the keys are cut by who holds them: the prefix of a group of rows (one range for all the group's
// queries) and each row's keys behind it.  All query heads of a kv head read the same keys, so a
// range's queries are its (token, head) pairs: column p of a tile is token p / group, head p % group.
// A prefix that costs more that way than every row by itself (rows whose own pairs fill tiles: sharing saves
// them no matrix products) is not shared (shared_keys).
//
// Ranges, and the work.  Range s < B is the prefix of the group that row s leads, range B + b row b's
// own keys.  A range of up to 32 pairs is narrow: its items (kv head) are walked by single waves, 64
// keys a unit.  A wider one is cut into tiles of up to 128 pairs, whose items (kv head, tile) are walked
// by whole work-groups, 128 keys a unit.  The units of each kind are dealt out in equal contiguous
// shares, over the work-groups (one of 8 waves per CU) and over their waves; every work-group finds its
// shares from the lengths, so a captured launch follows them.  A worker leaves its part of an item in
// the workspace, and shared_merge_kernel merges the parts of each (token, head).
//
// The walks.  K and V travel from memory to LDS (buffer_load ... lds); S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_32x32x16 as in the prefill kernel: one column per lane, P in registers as it comes.  K rows
// of 256 bytes with chunk ^ row % 16, V with chunk ^ 4 (row % 4), so that the reads of both (V's
// transposing) are free of bank conflicts.
//   A wide item's 128-key steps are loaded by all eight waves, one 16-key run each (a run lies in one
// block), a step ahead; a wave takes 32 columns and 64 keys of a step (up to 128 columns) or 32 keys (up
// to 64), and the key streams meet in LDS at the end.
//   A narrow item's 32-key steps are one wave's, in LDS of its own without barriers: once K is in
// registers the next step's K is sent for, likewise V.
//
// What bounds it.  A wide step takes about 4,300 cycles, of which the MFMAs are 2,048 on each SIMD and LDS is
// busy for 2,560 (3,700 without the loads); with all CUs at it 2.3 us at the 1.83 GHz they then hold, 930
// TFLOP/s.  A call costs about 10 us beside its steps: launch 2, plan 1.5, first loads and queries 2.5, the
// parts' way out 2, the merge 3 to 4.  Replayed at the clock of steady work, keys in the caches, 12 heads of 2
// kv heads: 2 rows of 100 keys 10.2 us (each row's keys read for it alone by the paged kernels: 6.6), 16 branches
// of 2,048 keys 15.0 (14.8; from memory 15.5 and 17.0), 40 rows in 9 groups (52 MB of keys) 20.8 (36.6), 12 rows of
// 1 to 17 new tokens over 3,001 keys 23.3 (41.5), 64 branches of 31,000 keys 38 (267), 8 rows of 90 to 150 new tokens
// over 5,000 keys and up to 900 of their own 54 (73): these share nothing, and gain by keys dealt out evenly.
// A prefix of several tiles is fetched into the L2s by each of them (64 branches of 31,000 keys: three tiles, 131
// MB, of which 65 are distinct; an XCD's share is less than one of the tiles, so they do not meet in its L2).
#include "cache_ops.h"

#include <type_traits>

namespace mi_fa2 {

constexpr int kShWaves = kSharedWaves, kShThreads = 64 * kShWaves;
constexpr int kShTile = kSharedTile;            // pairs of a wide tile
constexpr int kShNarrow = kSharedNarrow;        // pairs a narrow range has at most
constexpr int kShStep = 32;                     // keys of an MFMA block, and of a narrow step
constexpr int kShNarrowUnit = 64;
constexpr int kShWideUnit = 128;                // keys of a wide step
// What an item costs beside its units (queries, the first loads' latency, its part's way out), in units:
// it takes as many shares more, before its units.
constexpr int kShWideCost = 4, kShNarrowCost = 1;
constexpr int kShMergeCost = 4;   // of one more wide part for each pair, in the merge
constexpr int kShNarrowWeight = 7;
// Narrow shares go to as many work-groups as there is room for, a wave each, then a second wave of each: 64 keys
// that a wave has to itself arrive sooner than with seven more of its CU's (2 rows of 100 keys 11.1 -> 10.4
// us).  From kShSpread shares for each work-group on a wave takes kShEach, so that
// an item leaves fewer parts (40 rows in 9 groups, 52 MB, 24.6 -> 21.5 us; two each 22.7), or more where
// eight waves of each do not do, and no more waves than that takes (172 rows of 34 groups 30.9 -> 29.6).
constexpr int kShSpread = 4, kShEach = 3;
constexpr int kShRow = kHeadDim * 2;            // bytes of a key
constexpr int kShStage = 2 * kShWideUnit * kShRow;   // K, then V, of a wide step: 64 KB
constexpr int kShRing = 2 * kShStage / kShWaves;     // a wave's part of the two stages: 16 KB
static_assert(kShRing == 2 * kShStep * kShRow, "a narrow step's K and V");

// Tokens and keys of a range: keys [k0, k1) of the row's table (range s: row s, or s - B).
struct ShRange {
  int t0, tokens, k0, k1;
};

// What a work-group knows of the call, in LDS.
struct ShPlan {
  int wide[2 * kShMaxRows + 1];    // shares of the ranges before this one (see kShWideCost)
  int narrow[2 * kShMaxRows + 1];
  ShRange range[2 * kShMaxRows];
};

// What it is made from, where K and V will be.
struct ShRows {
  int cu[kShMaxRows + 1];          // as given, inside q
  int kv[kShMaxRows];
  int group[kShMaxRows];           // by group: first row and the row after its last, packed; -1: none
  int group_prefix[kShMaxRows];
  int mark[kShMaxRows];            // at a group's first row: which group, and the row after its last
  int t0[kShMaxRows], tokens[kShMaxRows];
  int lead[kShMaxRows];            // the first row of the row's group, -1: none
  // at a group's first row:
  int prefix[kShMaxRows];          // keys that each of its queries sees
  int last[kShMaxRows];            // the token after its last
  int alone[kShMaxRows];           // what 128 keys cost without sharing, in shares
};

// a / b of whole numbers >= 0, b > 0.  Below 2^22 by the reciprocal: the product is off by less than one.
__device__ __forceinline__ int quotient(int a, int b) {
  if (a >= 1 << 22 || b >= 1 << 22) return (unsigned)a / (unsigned)b;
  int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));
  const int r = a - q * b;
  q += r >= b ? 1 : r < 0 ? -1 : 0;
  return __builtin_amdgcn_readfirstlane(q);
}

__device__ __forceinline__ int wide_tiles(int pairs) { return (pairs + kShTile - 1) / kShTile; }
// pairs of a tile: the range's, evenly, in whole 32s
__device__ __forceinline__ int tile_pairs(int pairs, int tiles) {
  return (quotient(pairs + tiles - 1, tiles) + 31) & ~31;
}
__device__ __forceinline__ int key_units(const ShRange& r, int unit) {
  return max(1, (r.k1 - r.k0 + unit - 1) / unit);
}

__device__ __forceinline__ ShRange uniform(const ShRange& r) {
  return {__builtin_amdgcn_readfirstlane(r.t0), __builtin_amdgcn_readfirstlane(r.tokens),
          __builtin_amdgcn_readfirstlane(r.k0), __builtin_amdgcn_readfirstlane(r.k1)};
}

// Inclusive sum or maximum (of numbers >= 0) over the wave's lanes.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
template <bool MAX>
__device__ __forceinline__ int wave_scan(int x) {
  const auto op = [](int a, int b) { return MAX ? max(a, b) : a + b; };
  x = op(x, dpp<0x111, 0xf>(x));   // row_shr 1, 2, 4, 8: within 16 lanes
  x = op(x, dpp<0x112, 0xf>(x));
  x = op(x, dpp<0x114, 0xf>(x));
  x = op(x, dpp<0x118, 0xf>(x));
  x = op(x, dpp<0x142, 0xa>(x));   // lane 15 of a row to the next, lane 31 to the upper half
  return op(x, dpp<0x143, 0xc>(x));
}

// One wave's LDS accesses before this come before those after it.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The keys read once for the group that row `lead` leads: whole steps of its prefix, or none where that
// would cost more shares than every row by itself (one row; rows that fill tiles of their own, and then
// pay for another item each).
__device__ __forceinline__ int shared_keys(const SharedParams& p, const ShRows& rows, int lead) {
  const int keys = rows.prefix[lead] & ~(kShStep - 1);
  const int pairs = (rows.last[lead] - rows.t0[lead]) * p.group;
  const float blocks = (float)keys * (1.f / 128.f);
  const float shared =
      pairs > kShNarrow
          ? (float)(kShNarrowWeight * wide_tiles(pairs)) * (blocks + kShWideCost + kShMergeCost)
          : 2.f * blocks + kShNarrowCost;
  return shared < (float)rows.alone[lead] * blocks ? keys : 0;
}

// Everything by one wave, 64 rows at a time, so that it needs no barrier but one.
__device__ __forceinline__ void make_plan(const SharedParams& p, ShPlan& pl, ShRows& rows) {
  const int lane = threadIdx.x & 63, B = p.B;
  if (threadIdx.x < 64) {
    for (int b = lane; b <= B; b += 64) {
      const int c = p.cu_q[b], kv = b < B ? p.kv_lens[b] : 0;
      const int lo = b < p.G ? p.cu_rows[b] : 0, hi = b < p.G ? p.cu_rows[b + 1] : 0;
      const int shared = b < p.G ? p.prefix_lens[b] : 0;
      rows.cu[b] = clamp_len(c, p.total_q);
      if (b < B) {
        rows.kv[b] = clamp_len(kv, p.max_kv);
        rows.group[b] = lo >= 0 && lo < hi && hi <= B ? lo << 16 | hi : -1;
        rows.group_prefix[b] = clamp_len(shared, p.max_kv);
        rows.mark[b] = 0;
        rows.prefix[b] = p.max_kv;
        rows.last[b] = 0;
        rows.alone[b] = 0;
      }
    }
    wave_fence();
    // groups mark their first rows (of several with one first row, the last group counts)
    for (int g = lane; g < p.G; g += 64) {
      const int ends = rows.group[g];
      if (ends >= 0) atomicMax(&rows.mark[ends >> 16], (g + 1) << 10 | (ends & 0xffff));
    }
    wave_fence();
    // A row's group is that of the last first row up to it, if it reaches the row; offsets never fall.
    // Each row tells its group's first row what it sees, holds and costs.
    int first_top = 0, cu_top = 0;
    for (int base = 0; base < B; base += 64) {
      const int b = base + lane, at = min(b, B - 1);
      const int mark = b < B ? rows.mark[at] : 0, next = rows.cu[at + 1], kv = rows.kv[at];
      const int cu = max(cu_top, wave_scan<true>(b < B ? rows.cu[at] : 0));
      // first row + 1, group + 1, row after its last: ten bits each
      const int first = max(first_top, wave_scan<true>(mark ? (b + 1) << 20 | mark : 0));
      first_top = __builtin_amdgcn_readlane(first, 63);
      cu_top = __builtin_amdgcn_readlane(cu, 63);
      if (b < B) {
        const int lead = b < (first & 0x3ff) ? (first >> 20) - 1 : -1;
        const int tokens = max(next - cu, 0), pairs = tokens * p.group;
        rows.t0[b] = cu;
        rows.tokens[b] = tokens;
        rows.lead[b] = lead;
        if (lead >= 0) {
          int seen = tokens == 0 ? p.max_kv : max(0, p.causal ? kv - tokens + 1 : kv);
          // the first row has to hold the prefix
          if (lead == b) seen = min(seen, min(kv, rows.group_prefix[((first >> 10) & 0x3ff) - 1]));
          atomicMin(&rows.prefix[lead], seen);
          atomicMax(&rows.last[lead], cu + tokens);
          if (pairs > 0)
            atomicAdd(&rows.alone[lead], pairs > kShNarrow ? kShNarrowWeight * wide_tiles(pairs) : 2);
        }
      }
    }
    wave_fence();
    int wide_top = 0, narrow_top = 0;
    if (lane == 0) pl.wide[0] = pl.narrow[0] = 0;
    for (int base = 0; base < 2 * B; base += 64) {
      const int s = base + lane;
      int wide = 0, narrow = 0;
      if (s < 2 * B) {
        const int b = s < B ? s : s - B, lead = rows.lead[b];
        const int shared = lead >= 0 ? shared_keys(p, rows, lead) : 0;
        ShRange r = {rows.t0[b], rows.tokens[b], shared, rows.kv[b]};
        if (s < B) {
          r.tokens = lead == b && shared > 0 ? rows.last[b] - r.t0 : 0;
          r.k0 = 0;
          r.k1 = shared;
        }
        pl.range[s] = r;
        const int pairs = r.tokens * p.group;
        if (pairs > kShNarrow)
          wide = p.Hkv * wide_tiles(pairs) * (key_units(r, kShWideUnit) + kShWideCost);
        else if (pairs > 0)
          narrow = p.Hkv * (key_units(r, kShNarrowUnit) + kShNarrowCost);
      }
      wide = wide_top + wave_scan<false>(wide);
      narrow = narrow_top + wave_scan<false>(narrow);
      wide_top = __builtin_amdgcn_readlane(wide, 63);
      narrow_top = __builtin_amdgcn_readlane(narrow, 63);
      if (s < 2 * B) {
        pl.wide[s + 1] = wide;
        pl.narrow[s + 1] = narrow;
      }
    }
  }
  __syncthreads();
}

// The range that holds share u: R[s] <= u < R[s + 1] (0 <= u < R[n]), by a whole wave.
__device__ __forceinline__ int find_range(const int* R, int n, int u, int lane) {
  int at = -1;
  for (int base = 0; base < n; base += 64)
    at += __popcll(__ballot(base + lane < n && R[min(base + lane, n)] <= u));
  return __builtin_amdgcn_readfirstlane(at);
}

// N shares over W <= N workers: the first `rem` have q + 1, the others q.
struct ShDeal {
  int q, rem;
};
__device__ __forceinline__ ShDeal make_deal(int N, int W) {
  const int q = W > 0 ? quotient(N, W) : 0;
  return {q, N - q * W};
}
__device__ __forceinline__ int first_of(const ShDeal& d, int w) { return w * d.q + min(w, d.rem); }
__device__ __forceinline__ int worker_of(const ShDeal& d, int u) {
  const int big = d.rem * (d.q + 1);
  return u < big ? quotient(u, d.q + 1) : d.rem + quotient(u - big, d.q);
}

// The part of a walk that is the same for all its steps.
struct ShWalk {
  const int32_t* table;   // the row's block ids
  const uint16_t* k;      // pools at the kv head
  const uint16_t* v;
  int end;                // keys of the range end here: later rows read as zeros
  int full;               // keys before this are seen by every column
};

// One wave's 32 columns.
struct ShState {
  u32x4 q[8];             // queries: d = 16 s + 8 g + [0, 8)
  f32x16 o[4];            // accumulator r of block db: d = 32 db + 8 (r / 4) + 4 g + r % 4
  float m, l;             // running max (of the unscaled scores) and this lane's part of the sum
  int lim;                // keys before this are seen by the lane's column
};

// Lane's offsets in a 16-key run: load instruction j moves rows 4 j + lane / 16 to LDS chunk lane % 16, the
// chunk of K it takes being that ^ row, of V ^ 4 (row % 4).
struct ShLanes {
  int row, k, v;   // bytes: of row lane / 16, of the chunks in instruction 0
};
__device__ __forceinline__ ShLanes lane_offsets(int64_t kv_st, int lane) {
  const int row = lane >> 4;
  return {row * (int)kv_st * 2, 16 * ((lane & 15) ^ row), 16 * ((lane & 15) ^ (4 * row))};
}

// The block id of the 16 keys from t on.
__device__ __forceinline__ int entry_of(const SharedParams& p, const ShWalk& w, int64_t t) {
  return t < w.end ? w.table[t >> p.bs_shift] : -1;
}

// 16 keys of K or V from t on, in block blk: where they are; keys past the range's end are outside.
struct ShRun {
  uint64_t base;
  uint32_t bytes;
};
template <bool V>
__device__ __forceinline__ ShRun run_at(const SharedParams& p, const ShWalk& w, int blk, int t) {
  const bool in = (unsigned)blk < (unsigned)p.num_blocks;
  const int64_t slot = ((int64_t)(in ? blk : 0) << p.bs_shift) + (t & ((1 << p.bs_shift) - 1));
  const uint32_t bytes = in ? (uint32_t)(sclamp(w.end - t, 0, 16) * (int)p.kv_st * 2) : 0u;
  return {uniform_u64(reinterpret_cast<uint64_t>((V ? w.v : w.k) + slot * p.kv_st)),
          (uint32_t)__builtin_amdgcn_readfirstlane(bytes)};
}
// K runs of 64 steps, a lane each, found in a few vector instructions: the lane's first key is t.
struct ShRuns {
  uint32_t lo, hi, bytes;
};
__device__ __forceinline__ ShRuns find_runs(const SharedParams& p, const ShWalk& w, int64_t t, int blk) {
  const bool in = (unsigned)blk < (unsigned)p.num_blocks;
  const int64_t slot = ((int64_t)(in ? blk : 0) << p.bs_shift) + ((int)t & ((1 << p.bs_shift) - 1));
  const uint64_t at = reinterpret_cast<uint64_t>(w.k + slot * p.kv_st);
  const int rows = (int)min<int64_t>(max<int64_t>(w.end - t, 0), 16);
  return {(uint32_t)at, (uint32_t)(at >> 32), in ? (uint32_t)(rows * (int)p.kv_st * 2) : 0u};
}
__device__ __forceinline__ ShRun run_of(const ShRuns& runs, int lane) {
  return {(uint64_t)(uint32_t)__builtin_amdgcn_readlane(runs.hi, lane) << 32 |
              (uint32_t)__builtin_amdgcn_readlane(runs.lo, lane),
          (uint32_t)__builtin_amdgcn_readlane(runs.bytes, lane)};
}

// Load instruction j (0 .. 3) of a run to LDS; what is outside becomes zeros.
template <bool V>
__device__ __forceinline__ void load_rows(const SharedParams& p, const ShRun& run, int j, uint32_t lds,
                                          const ShLanes& ln) {
  const int row = opaque(ln.row);   // the sum is made here, not kept
  lds_dma16(run.base, run.bytes, lds + 1024 * j,
            row + j * 8 * (int)p.kv_st + (V ? ln.v : ln.k ^ (64 * j)));
}
template <bool V>
__device__ __forceinline__ void load_run(const SharedParams& p, const ShWalk& w, int blk, int t,
                                         uint32_t lds, const ShLanes& ln) {
  const ShRun run = run_at<V>(p, w, blk, t);
#pragma unroll
  for (int j = 0; j < 4; ++j) load_rows<V>(p, run, j, lds, ln);
}

// The operands of 32 keys out of LDS.  MFMA row r of S^T is key pi(r), so that a lane's 8 keys of a
// 16-key step are consecutive.
__device__ __forceinline__ int k_offset(int lane) {
  const int r32 = lane & 31, g = lane >> 5;
  const int pim = 16 * (r32 >> 4) + 8 * ((r32 >> 2) & 1) + 4 * ((r32 >> 3) & 1) + (r32 & 3);
  return pim * 256 + 16 * (g ^ (pim & 1)) + 32 * ((pim >> 1) & 7);
}
__device__ __forceinline__ void read_k(const uint8_t* k, int lane, u32x4 (&ka)[8]) {
  const int kx = k_offset(lane);
#pragma unroll
  for (int s = 0; s < 8; ++s) ka[s] = *reinterpret_cast<const u32x4*>(k + (kx ^ (32 * s)));
}
__device__ __forceinline__ u32x4 read_v(const uint8_t* v, int lane, int kk, int db) {
  const int g = lane >> 5, vk = (lane >> 2) & 3;
  const uint8_t* a = v + 2048 * g + 256 * vk + 32 * ((lane >> 4) & 1) + 8 * (lane & 3) +
                     64 * (db ^ vk) + 4096 * kk;
  const u32x2 lo = ds_read_tr16(a);
  const u32x2 hi = ds_read_tr16(a + 1024);
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

__device__ __forceinline__ void read_v(const uint8_t* v, int lane, u32x4 (&va)[2][4]) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int db = 0; db < 4; ++db) va[kk][db] = read_v(v, lane, kk, db);
}

// S^T of 32 keys and the wave's columns.
template <typename E>
__device__ __forceinline__ f32x16 scores(const u32x4 (&ka)[8], const u32x4 (&q)[8]) {
  f32x16 s = f32x16{};
#pragma unroll
  for (int k = 0; k < 8; ++k) s = E::mfma32(ka[k], q[k], s);
  return s;
}

// The same for N blocks of 32 keys in LDS, operands read two k-steps ahead of their MFMAs and no further.
// between(0 .. 3) is called between the MFMAs (the next step's loads), as in ShPv.
template <typename E, int N, typename F>
__device__ __forceinline__ void scores_of(const uint8_t* k, int lane, const u32x4 (&q)[8],
                                          f32x16 (&s)[N], F&& between) {
  const int kx = k_offset(lane);
  u32x4 ka[3][N];
  const auto rd = [&](int i) {
#pragma unroll
    for (int n = 0; n < N; ++n)
      ka[i % 3][n] = *reinterpret_cast<const u32x4*>(k + (kx ^ (32 * i)) + n * kShStep * kShRow);
  };
  rd(0);
  rd(1);
#pragma unroll
  for (int n = 0; n < N; ++n) s[n] = f32x16{};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i + 2 < 8) rd(i + 2);
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] = E::mfma32(ka[i % 3][n], q[i], s[n]);
    if (i & 1) between(i >> 1);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// O += P V of N blocks of 32 keys in LDS.  V's operands are read a k-step ahead, those of the first (begin)
// before the softmax or scores that come in between.
template <typename E, int N>
struct ShPv {
  u32x4 va[2][4];

  __device__ __forceinline__ void read(const uint8_t* v, int lane, int i) {
#pragma unroll
    for (int db = 0; db < 4; ++db)
      va[i & 1][db] = read_v(v + (i >> 1) * kShStep * kShRow, lane, i & 1, db);
  }
  __device__ __forceinline__ void begin(const uint8_t* v, int lane) {
    read(v, lane, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
  template <typename F>
  __device__ __forceinline__ void add(ShState& st, const uint8_t* v, int lane, const u32x4 (&pb)[2 * N],
                                      F&& between) {
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
      if (i + 1 < 2 * N) read(v, lane, i + 1);
#pragma unroll
      for (int db = 0; db < 4; ++db) st.o[db] = E::mfma32(va[i & 1][db], pb[i], st.o[db]);
#pragma unroll
      for (int j = 0; j < 2 / N; ++j) between(i * (2 / N) + j);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// Accumulator r of a block of 32 keys is the lane's key 16 (r / 8) + r % 8 (the lanes with g = 1 start at
// key 8): those at or past lim are hidden.
__device__ __forceinline__ void hide(f32x16& s, int lim) {
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (16 * (r >> 3) + (r & 7) >= lim) s[r] = -INFINITY;
}

// The online softmax of N blocks of 32 keys: P^T as the B operand (block n's 16-key step kk in pb[2 n +
// kk]), maximum, sum and O updated.
//   p = 2^(c (s - m)): the difference first, so that scores of any size keep their weights.  The
// reference m may lag the true maximum while no p of the lane exceeds 2^8, as in the prefill kernel.
// The first keys of a walk (fresh) have no reference yet.
//   P is rounded to the 16-bit type, as the MFMA takes it and as the other attention kernels here do; the
// sum is of the rounded values, so that the weights still add up to one.  In bf16 the output is then 0.0021 to
// 0.0023 of its size off from 64 bits, 0.0017 with P in 32 bits (the rounding of the output alone).
template <typename E, int N>
__device__ __forceinline__ void softmax(float c, ShState& st, const f32x16 (&s)[N], u32x4 (&pb)[2 * N],
                                        bool fresh) {
  const auto weigh = [&](float ref) {
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t x =
            E::pack2(exp2_fast((s[n][2 * i] - ref) * c), exp2_fast((s[n][2 * i + 1] - ref) * c));
        pb[2 * n + (i >> 2)][i & 3] = x;
        sum = E::sum2(x, sum);
      }
    return sum;
  };
  float sum = INFINITY;
  if (!fresh) sum = weigh(st.m);
  if (__any(!(sum <= 256.f))) {
    float mx = -INFINITY;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[n][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const bool grow = (mx - st.m) * c > 8.f;
    if (fresh) {   // nothing to rescale
      st.m = mx;
    } else if (__any(grow)) {
      const float alpha = grow ? exp2_fast((st.m - mx) * c) : 1.f;
      st.l *= alpha;
#pragma unroll
      for (int i = 0; i < 4; ++i) st.o[i] *= alpha;
      if (grow) st.m = mx;
    }
    sum = weigh(st.m == -INFINITY ? 0.f : st.m);
  }
  st.l += sum;
}

// O += P V of 32 keys.
template <typename E>
__device__ __forceinline__ void add_pv(ShState& st, const u32x4 (&va)[2][4], const u32x4* pb) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int db = 0; db < 4; ++db) st.o[db] = E::mfma32(va[kk][db], pb[kk], st.o[db]);
}

// Whether N blocks of 32 keys in LDS hold a value that is inf or NaN: all its exponent bits set, which a 1
// added to the exponent carries into the sign's place.
template <typename E, int N>
__device__ __forceinline__ bool any_odd(const uint8_t* v, int lane) {
  constexpr uint32_t kMant = E::kOnes2 == 0x3f803f80u ? 0x007f007fu : 0x03ff03ffu;
  constexpr uint32_t kUnit = kMant + 0x00010001u, kExp = 0x7fff7fffu & ~kMant;
  uint32_t odd = 0;
  lane = opaque(lane);   // rare: its addresses are not kept through the key loop
#pragma unroll 2
  for (int i = 0; i < 8 * N; ++i) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(v + 1024 * i + 16 * lane);
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= ((x[e] & kExp) + kUnit) & 0x80008000u;
  }
  return __any(odd != 0);
}

// The wave's columns [col0, col0 + 32) of a tile of `cols` that begins with pair `pair0` of the range.
__device__ __forceinline__ void start_tile(const SharedParams& p, const ShRange& r, bool own, int hk,
                                           int pair0, int col0, int cols, int lane, ShWalk& w,
                                           ShState& st) {
  const int g = lane >> 5, col = col0 + (lane & 31);
  // own keys: query i of the row's n sees all but the n - 1 - i last
  const int first = r.k1 - r.tokens + 1;
  const int token = fdiv(pair0 + col, p.group_div);
  w.full = own && p.causal ? min(r.k1, first + fdiv(pair0 + col0, p.group_div)) : r.k1;
  st.lim = own && p.causal ? min(r.k1, first + token) : r.k1;
  if (col < cols) {
    const uint16_t* q = p.q + (int64_t)(r.t0 + token) * p.q_st +
                        (int64_t)(hk * p.group + (pair0 + col - token * p.group)) * p.q_sh + 8 * g;
#pragma unroll
    for (int s = 0; s < 8; ++s) st.q[s] = ld16(q + 16 * s);
  } else {
#pragma unroll
    for (int s = 0; s < 8; ++s) st.q[s] = u32x4{0, 0, 0, 0};
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) st.o[i] = f32x16{};
  st.m = -INFINITY;
  st.l = 0.f;
}

// Where the parts of the item's pairs stand: written by the worker with the item's first unit.  The
// record of a pair: its first part's column, and the number of parts with the kind of worker and, for a
// row's own range, whether the row's group has a prefix.
__device__ __forceinline__ void record(const SharedParams& p, const ShRange& r, bool own, bool wide,
                                       int hk, int pair, int column, int parts) {
  const int token = fdiv(pair, p.group_div);
  const int at = ((own ? p.total_q : 0) + r.t0 + token) * p.Hq + hk * p.group + (pair - token * p.group);
  const bool prefix = own && r.k0 > 0;
  *reinterpret_cast<int2*>(p.ws_where + 2 * (int64_t)at) =
      int2{column, parts << 2 | (wide ? 2 : 0) | (prefix ? 1 : 0)};
}

// Columns before the parts of an item's pairs (its kind's workers add theirs).
__device__ __forceinline__ int item_columns(const SharedParams& p, const ShRange& r, bool own, int hk,
                                            int pair0) {
  return ((own ? p.total_q : 0) + r.t0) * p.Hq + hk * r.tokens * p.group + pair0;
}

// Keys [kb, stop) of a tile's columns, one column a wave at a time, two dims a lane: for items some of
// whose values are not finite and hidden from some of their queries, where the product of a whole tile
// would have 0 x inf.  A hidden key is not looked at here.
template <typename E>
__device__ __forceinline__ void careful_item(const SharedParams& p, const ShRange& r, int row, bool own,
                                             int hk, int pair0, int cols, int kb, int stop, int column, int wave,
                                             int waves, int lane) {
  lane = opaque(lane);
  const float c = p.scale_log2;
  const int32_t* table = p.table + row * p.bt_stride;
  for (int col = wave; col < cols; col += waves) {
    const int token = fdiv(pair0 + col, p.group_div), h = pair0 + col - token * p.group;
    const int lim = min(stop, own && p.causal ? r.k1 - r.tokens + 1 + token : r.k1);
    const uint32_t q = *reinterpret_cast<const uint32_t*>(
        p.q + (int64_t)(r.t0 + token) * p.q_st + (int64_t)(hk * p.group + h) * p.q_sh + 2 * lane);
    float m = -INFINITY, l = 0.f, oa = 0.f, ob = 0.f;
    for (int t = kb; t < lim; ++t) {
      const int blk = table[t >> p.bs_shift];
      const bool in = (unsigned)blk < (unsigned)p.num_blocks;
      const int64_t slot = ((int64_t)(in ? blk : 0) << p.bs_shift) + (t & ((1 << p.bs_shift) - 1));
      const int64_t at = slot * p.kv_st + hk * p.kv_sh + 2 * lane;
      const uint32_t k = in ? *reinterpret_cast<const uint32_t*>(p.k + at) : 0;
      const uint32_t v = in ? *reinterpret_cast<const uint32_t*>(p.v + at) : 0;
      float s = E::lo(q) * E::lo(k) + E::hi(q) * E::hi(k);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
      const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn;
      const float a = exp2_fast((m - mu) * c), w = exp2_fast((s - mu) * c);
      l = l * a + w;
      oa = oa * a + w * E::lo(v);
      ob = ob * a + w * E::hi(v);
      m = mn;
    }
    float* o = p.ws_o + (int64_t)(column + col) * kHeadDim + 2 * lane;
    o[0] = oa;
    o[1] = ob;
    if (lane == 0) {
      p.ws_ml[2 * (int64_t)(column + col)] = m;
      p.ws_ml[2 * (int64_t)(column + col) + 1] = l;
    }
  }
}

// Units [c0, c1) of a wide item by the work-group: RG blocks of 32 columns, 8 / RG key streams, a unit a
// step.  Waves w and w + 4 share a SIMD and take keys of a step's two halves half a step apart, so that one's
// softmax runs beside the other's MFMAs:
//   first half, step j:  softmax(j), O += PV(j), S(j + 1)      second half:  S(j), O += PV(j - 1), softmax(j)
// (S(0) comes before both).
// Slot j % 2 of the ring therefore holds, in step j, of the first half V(j) and K(j + 1), of the second K(j)
// and V(j - 1); it is loaded during step j - 1, each wave its run of either.
template <typename E, int RG>
__device__ __forceinline__ void wide_item(const SharedParams& p, const ShRange& r, int row, bool own,
                                          int hk, int pair0, int cols, int c0, int c1, int column, uint8_t* ring,
                                          float (*ml)[32][2], int* odd) {
  constexpr int KS = kShWaves / RG, N = kShWideUnit / KS / kShStep;   // 32-key blocks of a wave and step
  // (the lane as a value of this item: its many LDS addresses are not kept from one to the next)
  const int tid = threadIdx.x, lane = opaque(tid & 63);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = wave % RG, ks = wave / RG;
  const bool second = wave >= kShWaves / 2;
  const int g = lane >> 5;
  const int first = r.k0 + c0 * kShWideUnit, n = c1 - c0;
  ShWalk w;
  ShState st;
  w.table = p.table + row * p.bt_stride;
  w.k = p.k + hk * p.kv_sh;
  w.v = p.v + hk * p.kv_sh;
  w.end = r.k1;
  // this wave's run of step i: keys first + 128 i + 16 wave ..  (The first block ids travel while the
  // queries are found.)
  const auto run_key = [&](int i) { return first + (i + (int64_t)lane) * kShWideUnit + 16 * wave; };
  const int entry = entry_of(p, w, run_key(0));
  start_tile(p, r, own, hk, pair0, 32 * rg, cols, lane, w, st);
  const bool active = 32 * rg < cols;
  if (tid == 0) *odd = 0;   // (barriers follow)
  const ShLanes ln = lane_offsets(p.kv_st, lane);
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_addr_of(ring)) + wave * 16 * kShRow;
  constexpr uint32_t kV = kShWideUnit * kShRow;   // V of a slot, behind K
  ShRuns runs = find_runs(p, w, run_key(0), entry);
  const uint64_t v_apart = uniform_u64(reinterpret_cast<uint64_t>(w.v) - reinterpret_cast<uint64_t>(w.k));
  int ahead = 0;                    // the step whose K run is next_k, and V run v_of(next_k)
  ShRun next_k = run_of(runs, 0), next_v{};
  const auto v_of = [&](const ShRun& k) { return ShRun{k.base + v_apart, k.bytes}; };
  const auto step_ahead = [&]() {
    ++ahead;
    if ((ahead & 63) == 0) runs = find_runs(p, w, run_key(ahead), entry_of(p, w, run_key(ahead)));
    next_k = run_of(runs, ahead & 63);
  };
  const auto load_all = [&](auto v, const ShRun& run, uint32_t at) {
#pragma unroll
    for (int i = 0; i < 4; ++i) load_rows<decltype(v)::value>(p, run, i, at, ln);
  };
  constexpr std::false_type isK{};
  constexpr std::true_type isV{};
  if (!second) {
    load_all(isK, next_k, lds + kShStage);
    load_all(isV, v_of(next_k), lds + kV);
    if (n > 1) {
      step_ahead();
      load_all(isK, next_k, lds);
    }
  } else {
    load_all(isK, next_k, lds);
    load_all(isV, v_of(next_k), lds + kShStage + kV);
  }
  const auto step_ready = [&]() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  // The loads of step j, for slot (j + 1) % 2, between the MFMAs: V of the last step whose K went out, K of
  // the next (the second half's first V came with the first loads).
  bool more_k = false, more_v = false;
  uint32_t next_lds = 0;
  const auto plan_loads = [&](int j) {
    next_lds = lds + ((j + 1) & 1) * kShStage;
    more_v = second ? j > 0 : j + 1 < n;
    next_v = v_of(next_k);
    more_k = ahead + 1 < n;
    if (more_k) step_ahead();
  };
  const auto load_k = [&](int i) {
    if (more_k) load_rows<false>(p, next_k, i, next_lds, ln);
  };
  const auto load_v = [&](int i) {
    if (more_v) load_rows<true>(p, next_v, i, next_lds + kV, ln);
  };

  const int offset = ks * N * kShStep;   // the stream's keys in a step
  const auto has = [&](int j) { return active && j < n && first + j * kShWideUnit + offset < w.end; };
  f32x16 s[N];
  u32x4 pb[2 * N];
  const auto do_scores = [&](int j, int slot, auto&& between) {
    if (has(j)) {
      scores_of<E, N>(ring + slot * kShStage + offset * kShRow, lane, st.q, s, between);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) between(i);
    }
  };
  const auto do_softmax = [&](int j) {
    if (!has(j)) return;
    const int kb = first + j * kShWideUnit + offset;
    if (kb + N * kShStep > w.full) {
#pragma unroll
      for (int b = 0; b < N; ++b) hide(s[b], st.lim - kb - kShStep * b - 8 * g);
    }
    softmax<E, N>(p.scale_log2, st, s, pb, j == 0);
  };
  ShPv<E, N> pv;
  const auto v_in = [&](int slot) { return ring + slot * kShStage + kV + offset * kShRow; };
  const auto begin_pv = [&](int j, int slot) {
    if (has(j)) pv.begin(v_in(slot), lane);
  };
  const auto do_pv = [&](int j, int slot, auto&& between) {
    if (has(j)) {
      const uint8_t* v = v_in(slot);
      if (first + j * kShWideUnit + offset + N * kShStep > w.full && any_odd<E, N>(v, lane)) *odd = 1;
      pv.add(st, v, lane, pb, between);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) between(i);
    }
  };
  // (The first half's K goes out with its V: behind its scores, the step's last, it would be waited for.  8 x 150
  // tokens over 5,000 keys 59.6 -> 58.4 us, 64 over 31,000 39.9 -> 39.1.)
  const auto none = [](int) {};
  const auto load_both = [&](int i) {
    load_k(i);
    load_v(i);
  };
  step_ready();
  // (separate programs of the same barriers)
  if (!second) {
    do_scores(0, 1, none);
    __syncthreads();
    for (int j = 0; j < n; ++j) {
      plan_loads(j);
      begin_pv(j, j & 1);
      do_softmax(j);
      do_pv(j, j & 1, load_both);
      do_scores(j + 1, j & 1, none);
      step_ready();
    }
  } else {
    do_scores(0, 0, none);
    __syncthreads();
    plan_loads(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) load_k(i);
    do_softmax(0);
    step_ready();
    for (int j = 1; j < n; ++j) {
      plan_loads(j);
      begin_pv(j - 1, j & 1);
      do_scores(j, j & 1, load_k);
      do_pv(j - 1, j & 1, load_v);
      do_softmax(j);
      step_ready();
    }
    begin_pv(n - 1, n & 1);
    do_pv(n - 1, n & 1, none);
  }
  // The key streams' parts become one.  A wave keeps 4 / KS of its four blocks of dims, gives the others away
  // through LDS, in the accumulators' order, and adds what it gets.
  st.l += __shfl_xor(st.l, 32);
  const int out_lane = opaque(lane), r32 = out_lane & 31;
  if (g == 0) {
    ml[wave][r32][0] = st.m;
    ml[wave][r32][1] = st.l;
  }
  constexpr int kKeep = 4 / KS;
  // The second half's waves may still read V of the last step (the last quarter of slot n % 2): the first
  // half writes to the other slot, the second to the first three quarters of that one.
  const auto area = [&](int wv, int db) {
    const int i = KS == 2 ? db & 1 : db - (db > wv / RG ? 1 : 0);   // of the blocks that the wave gives
    return ring + ((n + (wv < kShWaves / 2 ? 1 : 0)) & 1) * kShStage + (wv & 3) * 12288 + i * 4096 +
           out_lane * 16;
  };
#pragma unroll
  for (int db = 0; db < 4; ++db) {
    if (db / kKeep == ks) continue;   // (uniform)
#pragma unroll
    for (int rr = 0; rr < 4; ++rr)
      *reinterpret_cast<f32x4*>(area(wave, db) + rr * 1024) =
          f32x4{st.o[db][4 * rr], st.o[db][4 * rr + 1], st.o[db][4 * rr + 2], st.o[db][4 * rr + 3]};
  }
  __syncthreads();
  if (*odd) {
    careful_item<E>(p, r, row, own, hk, pair0, cols, first, min(r.k1, first + n * kShWideUnit), column, wave,
                    kShWaves, lane);
    __syncthreads();
    return;
  }
  float M = -INFINITY, L = 0.f, f[KS];
#pragma unroll
  for (int j = 0; j < KS; ++j) M = fmaxf(M, ml[j * RG + rg][r32][0]);
#pragma unroll
  for (int j = 0; j < KS; ++j) {
    f[j] = exp2_fast((ml[j * RG + rg][r32][0] - (M == -INFINITY ? 0.f : M)) * p.scale_log2);
    L = __builtin_fmaf(ml[j * RG + rg][r32][1], f[j], L);
  }
  const int col = 32 * rg + r32;
  float* o = p.ws_o + (int64_t)(column + col) * kHeadDim + 4 * g;
#pragma unroll
  for (int db = 0; db < 4; ++db) {
    if (db / kKeep != ks) continue;
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KS; ++j) {   // in the streams' order, whoever adds
        const f32x4 x = j == ks ? f32x4{st.o[db][4 * rr], st.o[db][4 * rr + 1], st.o[db][4 * rr + 2],
                                        st.o[db][4 * rr + 3]}
                                : *reinterpret_cast<const f32x4*>(area(j * RG + rg, db) + rr * 1024);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(x[e], f[j], sum[e]);
      }
      if (col < cols) *reinterpret_cast<f32x4*>(o + 32 * db + 8 * rr) = sum;
    }
  }
  if (ks == 0 && g == 0 && col < cols) {
    p.ws_ml[2 * (int64_t)(column + col)] = M;
    p.ws_ml[2 * (int64_t)(column + col) + 1] = L;
  }
  __syncthreads();   // the ring and ml are the next item's
}

// Keys [kb, stop) of a narrow item by one wave, in its own 16 KB of LDS.  Returns whether careful_item
// has to do it.
template <typename E>
__device__ __forceinline__ bool narrow_walk(const SharedParams& p, const ShWalk& w, ShState& st, int kb,
                                            int stop, int entry, const uint8_t* ring, int lane) {
  if (kb >= stop) return false;
  bool odd = false;
  const uint32_t lds_k = __builtin_amdgcn_readfirstlane(lds_addr_of(ring));
  const uint32_t lds_v = lds_k + kShStep * kShRow;
  const ShLanes ln = lane_offsets(p.kv_st, lane);
  int tbl = entry;   // block ids of the two runs of 32 steps, lane 2 i + run
  const auto load_k = [&](int i, int t) {
    load_run<false>(p, w, __builtin_amdgcn_readlane(tbl, 2 * i), t, lds_k, ln);
    load_run<false>(p, w, __builtin_amdgcn_readlane(tbl, 2 * i + 1), t + 16, lds_k + 16 * kShRow, ln);
  };
  const auto load_v = [&](int i, int t) {
    load_run<true>(p, w, __builtin_amdgcn_readlane(tbl, 2 * i), t, lds_v, ln);
    load_run<true>(p, w, __builtin_amdgcn_readlane(tbl, 2 * i + 1), t + 16, lds_v + 16 * kShRow, ln);
  };
  // the last item's reads have left LDS
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  load_k(0, kb);
  load_v(0, kb);
  for (int i = 1; kb < stop; ++i, kb += kShStep) {
    const int next = kb + kShStep;
    const bool more = next < stop;
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");   // K is there, V may be on its way
    u32x4 ka[8];
    read_k(ring, lane, ka);
    int ids = tbl;
    if (more) {
      if ((i & 31) == 0) ids = entry_of(p, w, next + (int64_t)lane * 16);
      tbl = ids;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // K has left LDS
      load_k(i & 31, next);
    }
    f32x16 s[1] = {scores<E>(ka, st.q)};
    const int g = lane >> 5;
    const bool masked = next > w.full;
    if (masked) hide(s[0], st.lim - kb - 8 * g);
    u32x4 pb[2];
    softmax<E, 1>(p.scale_log2, st, s, pb, i == 1);
    if (more)
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");   // V is there, the next K may be on its way
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const uint8_t* v = ring + kShStep * kShRow;
    if (masked) odd |= any_odd<E, 1>(v, lane);
    u32x4 va[2][4];
    read_v(v, lane, va);
    if (more) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // V has left LDS
      load_v(i & 31, next);
    }
    add_pv<E>(st, va, pb);
  }
  return odd;
}

template <typename E>
__global__ __launch_bounds__(kShThreads, 2) void shared_attn_kernel(const SharedParams p) {
  __shared__ __attribute__((aligned(1024))) uint8_t ring[kShWaves * kShRing];
  __shared__ ShPlan pl;
  __shared__ float ml[kShWaves][32][2];
  __shared__ int odd;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  make_plan(p, pl, *reinterpret_cast<ShRows*>(ring));
  const int n_ranges = 2 * p.B, W = gridDim.x;
  const int N1 = __builtin_amdgcn_readfirstlane(pl.wide[n_ranges]);
  const int N2 = __builtin_amdgcn_readfirstlane(pl.narrow[n_ranges]);
  // The wide ranges take the first W1 work-groups, the waves of the others the narrow ones: a share each
  // if that fits, else as many as their work weighs (a work-group's wide share takes 2.3 to 2.7 us, one of
  // eight narrow ones side by side 0.4: kShNarrowWeight of them are one; 5 to 9 differ by 1 %).
  int room = W - N1;
  if (N1 + (N2 + kShWaves - 1) / kShWaves > W) {
    const float all = (float)kShNarrowWeight * (float)N1 + (float)N2;
    room = min((N2 + kShWaves - 1) / kShWaves, (int)((float)W * (float)N2 / all + 0.5f));
    room = __builtin_amdgcn_readfirstlane(min(max(room, N2 > 0 ? 1 : 0), N1 > 0 ? W - 1 : W));
  }
  int W2 = N2;
  if (N2 > kShSpread * room) W2 = quotient(N2 - 1, max(kShEach, quotient(N2 - 1, kShWaves * room) + 1)) + 1;
  const int W3 = min(room, W2);
  const int W1 = min(W - W3, N1);

  if ((int)blockIdx.x < W1) {
    // work-group w runs on XCD w % 8: XCD x takes the x-th contiguous share of the work, so that its L2 holds what
    // its share reads.  (Tiles of one range meet in an L2 only if the share holds more than one of them.)
    const int x = blockIdx.x & 7, wg = x * (W1 >> 3) + min(x, W1 & 7) + ((int)blockIdx.x >> 3);
    const ShDeal deal = make_deal(N1, W1);
    int u = first_of(deal, wg);
    const int stop = first_of(deal, wg + 1);
    int s = find_range(pl.wide, n_ranges, u, lane);
    while (u < stop) {
      while (pl.wide[s + 1] <= u) ++s;
      s = __builtin_amdgcn_readfirstlane(s);
      const ShRange r = uniform(pl.range[s]);
      const bool own = s >= p.B;
      const int row = own ? s - p.B : s;
      const int pairs = r.tokens * p.group, tiles = wide_tiles(pairs), width = tile_pairs(pairs, tiles);
      const int units = key_units(r, kShWideUnit), length = units + kShWideCost;
      const int at = u - __builtin_amdgcn_readfirstlane(pl.wide[s]);
      const int item = quotient(at, length), pos = at - item * length;
      const int hk = quotient(item, tiles), pair0 = (item - hk * tiles) * width;
      const int take = min(length - pos, stop - u);
      const int c0 = max(0, pos - kShWideCost), c1 = pos + take - kShWideCost;
      if (c0 < c1) {
        const int cols = min(width, pairs - pair0);
        const int column = item_columns(p, r, own, hk, pair0) + wg * kShTile;
        if (c0 == 0 && tid < cols)
          record(p, r, own, true, hk, pair0 + tid, column + tid,
                 worker_of(deal, u + length - pos - 1) - wg + 1);
        if (cols <= 64)
          wide_item<E, 2>(p, r, row, own, hk, pair0, cols, c0, c1, column, ring, ml, &odd);
        else
          wide_item<E, 4>(p, r, row, own, hk, pair0, cols, c0, c1, column, ring, ml, &odd);
      }
      u += take;
    }
    return;
  }

  // neighbouring shares on different work-groups: a short list of units spreads over the CUs
  const int worker = wave * W3 + (int)blockIdx.x - (W - W3);
  if ((int)blockIdx.x < W - W3 || worker >= W2) return;
  const ShDeal deal = make_deal(N2, W2);
  int u = first_of(deal, worker);
  const int stop = first_of(deal, worker + 1);
  int s = find_range(pl.narrow, n_ranges, u, lane);
  while (u < stop) {
    while (pl.narrow[s + 1] <= u) ++s;
    s = __builtin_amdgcn_readfirstlane(s);
    const ShRange r = uniform(pl.range[s]);
    const bool own = s >= p.B;
    const int row = own ? s - p.B : s;
    const int pairs = r.tokens * p.group;
    const int length = key_units(r, kShNarrowUnit) + kShNarrowCost;
    const int at = u - __builtin_amdgcn_readfirstlane(pl.narrow[s]);
    const int hk = quotient(at, length), pos = at - hk * length;
    const int take = min(length - pos, stop - u);
    const int c0 = max(0, pos - kShNarrowCost), c1 = pos + take - kShNarrowCost;
    u += take;
    if (c0 >= c1) continue;
    const int column = p.narrow_base + item_columns(p, r, own, hk, 0) + worker * kShNarrow;
    if (c0 == 0 && lane < pairs)
      record(p, r, own, false, hk, lane, column + lane,
             worker_of(deal, u - take + length - pos - 1) - worker + 1);
    ShWalk w;
    ShState st;
    w.table = p.table + row * p.bt_stride;
    w.k = p.k + hk * p.kv_sh;
    w.v = p.v + hk * p.kv_sh;
    w.end = r.k1;
    const int kb = r.k0 + c0 * kShNarrowUnit, last = min(r.k1, r.k0 + c1 * kShNarrowUnit);
    const int entry = entry_of(p, w, kb + (int64_t)lane * 16);   // (travels while the queries are found)
    start_tile(p, r, own, hk, 0, 0, pairs, lane, w, st);
    if (narrow_walk<E>(p, w, st, kb, last, entry, ring + wave * kShRing, lane)) {
      careful_item<E>(p, r, row, own, hk, 0, pairs, kb, last, column, 0, 1, lane);
      continue;
    }
    const int r32 = lane & 31, g = lane >> 5;
    const float l = st.l + __shfl_xor(st.l, 32);
    if (r32 < pairs) {
      float* o = p.ws_o + (int64_t)(column + r32) * kHeadDim + 4 * g;
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
          *reinterpret_cast<f32x4*>(o + 32 * db + 8 * rr) =
              f32x4{st.o[db][4 * rr], st.o[db][4 * rr + 1], st.o[db][4 * rr + 2],
                    st.o[db][4 * rr + 3]};
      if (g == 0) {
        p.ws_ml[2 * (int64_t)(column + r32)] = st.m;
        p.ws_ml[2 * (int64_t)(column + r32) + 1] = l;
      }
    }
  }
}

// Merges the parts of one (token, head), by WAVES waves, or each half wave its own (WAVES = 0): every lane
// first takes a part's (m, l), as many parts a time as there are lanes, then a half wave its share of the
// parts' O, four dims a lane.  Bound by latency: the launch and two dependent reads, the record, then (m, l)
// and O: 4 us for 24 pairs of 2 parts, 6 us for 768 pairs of 44 (16 MB).  (The record, the weights and O one
// after the other: 25.1 us in all for 12 tokens over 3,001 keys instead of 23.6.)
template <typename E, int WAVES>
__global__ __launch_bounds__(256) void shared_merge_kernel(const SharedParams p) {
  constexpr int kLanes = WAVES > 0 ? 64 : 32;            // that weigh a pair's parts
  constexpr int kHalves = WAVES > 0 ? 2 * WAVES : 1;     // half waves that share them
  constexpr int kFlight = 4;                             // 2 to 8 differ by 2 %
  const int lane = threadIdx.x & 63, half = lane >> 5, d = 4 * (lane & 31);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = WAVES > 0 ? wave : 0, apart = WAVES > 0 ? half : 0;
  const int pair = WAVES > 0 ? (int)blockIdx.x : (int)blockIdx.x * 8 + 2 * wave + half;
  static_assert(WAVES == 0 || WAVES == 4, "a work-group's waves");
  if (pair >= p.total_q * p.Hq) return;
  const int token = fdiv(pair, p.heads_div), h = pair - token * p.Hq;
  const int32_t* where = p.ws_where + 2 * (int64_t)pair;
  const int64_t pairs = 2 * (int64_t)p.total_q * p.Hq;
  const int first = p.cu_q[0], last = p.cu_q[p.B];
  int col[2] = {where[0], where[pairs]}, n[2] = {where[1], where[pairs + 1]}, stride[2];
  const bool prefix = n[1] & 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    stride[i] = n[i] & 2 ? kShTile : kShNarrow;
    n[i] >>= 2;
  }
  if (!prefix) col[0] = n[0] = 0;
  // Tokens of no row have no record, and offsets that fall leave such tokens between the rows: whatever
  // stands there is not followed out of the workspace.
  if (token < first || token >= last) return;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (col[i] < 0 || n[i] < 0 || col[i] + ((int64_t)n[i] - 1) * stride[i] >= p.columns) return;

  const float c = p.scale_log2;
  const auto column = [&](int t) {
    return t < n[0] ? col[0] + (int64_t)t * stride[0] : col[1] + (int64_t)(t - n[0]) * stride[1];
  };
  float M = -INFINITY, L = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const int total = n[0] + n[1];
  for (int base = 0; base < total; base += kLanes) {
    const int i = base + (lane & (kLanes - 1)), batch = min(kLanes, total - base);
    const float2 part_ml = i < total ? *reinterpret_cast<const float2*>(p.ws_ml + 2 * (int64_t)column(i))
                                     : float2{-INFINITY, 0.f};
    // The first parts' O travels while what they weigh is found.
    f32x4 x[kFlight];
    const auto send = [&](int j0) {
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const int j = j0 + kHalves * k + apart;
        x[k] = j < batch ? *reinterpret_cast<const f32x4*>(p.ws_o + column(base + j) * kHeadDim + d)
                         : f32x4{0.f, 0.f, 0.f, 0.f};
      }
    };
    send(2 * part);
    const float m = part_ml.x, l = part_ml.y;
    float Mn = m;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) Mn = fmaxf(Mn, __shfl_xor(Mn, o));
    Mn = fmaxf(Mn, M);
    const float Mu = Mn == -INFINITY ? 0.f : Mn;
    const float old = exp2_fast((M - Mu) * c);
    // A part that saw no key (l is 0) doesn't count: its O may be anything.  One whose scores are NaN has a
    // maximum of -inf like it, but an l of NaN, and counts, whatever the others weigh.
    const float f = l == 0.f ? -1.f : exp2_fast((m - Mu) * c);
    float ls = l * f;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ls += __shfl_xor(ls, o);
    L = L * old + ls;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= old;
    M = Mn;
    for (int j0 = 2 * part; j0 < batch;) {   // (a wave's lanes stay together: they read each other's f)
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const int j = j0 + kHalves * k + apart;
        const float wt = __shfl(f, (lane & ~(kLanes - 1)) | (j & (kLanes - 1)));
        const bool live = j < batch && !(wt < 0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = live ? __builtin_fmaf(x[k][e], wt, acc[e]) : acc[e];
      }
      j0 += kHalves * kFlight;
      if (j0 < batch) send(j0);
    }
  }
  if constexpr (WAVES > 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], 32);
    __shared__ f32x4 sums[WAVES][32];
    if (half == 0) sums[part][lane] = acc;
    __syncthreads();   // (the whole block has one pair)
    if (part != 0 || half != 0) return;
#pragma unroll
    for (int j = 1; j < WAVES; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += sums[j][lane & 31][e];
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<u32x2*>(p.o + (int64_t)token * p.o_st + (int64_t)h * p.o_sh + d) =
      u32x2{E::pack2(acc[0] * inv, acc[1] * inv), E::pack2(acc[2] * inv, acc[3] * inv)};
  if (p.lse && (lane & 31) == 0)
    p.lse[h * p.l_sh + token * p.l_st] =
        L == 0.f ? -INFINITY : (M * c + __builtin_log2f(L)) * kLn2;
}

// From this many pairs on, half a wave merges each (fewer leave most of the device idle, and have more parts
// each): 1,032 pairs of 60 narrow parts 29.0 us in all by halves and 26.7 by four waves, 1,152 and 1,440 100.3 /
// 99.4 and 29.4 / 28.8, 2,048 34.2 / 35.6, 2,064 30.7 / 31.6, 4,080 35.7 / 39.5.
constexpr int kShMergePairs = 2048;

template <typename E>
static hipError_t launch_shared_t(const SharedParams& p, int n_wg, hipStream_t stream) {
  hipLaunchKernelGGL((shared_attn_kernel<E>), dim3(n_wg), dim3(kShThreads), 0, stream, p);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const int pairs = p.total_q * p.Hq;
  if (pairs < kShMergePairs)
    hipLaunchKernelGGL((shared_merge_kernel<E, 4>), dim3(pairs), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((shared_merge_kernel<E, 0>), dim3((pairs + 7) / 8), dim3(256), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_shared(SharedParams p, int dtype, int n_cus, void* workspace, hipStream_t stream) {
  const SharedSpace s = shared_space(p.total_q, p.Hq);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.ws_o = reinterpret_cast<float*>(ws);
  p.ws_ml = reinterpret_cast<float*>(ws + s.ml);
  p.ws_where = reinterpret_cast<int32_t*>(ws + s.where);
  p.columns = s.columns;
  p.narrow_base = s.narrow;
  p.group_div = make_fastdiv(p.group);
  p.heads_div = make_fastdiv(p.Hq);
  // (two at least: one for either kind of range)
  const int n_wg = n_cus < 2 ? 2 : n_cus < kSharedWgs ? n_cus : kSharedWgs;
  return dtype == 0 ? launch_shared_t<BF16>(p, n_wg, stream) : launch_shared_t<FP16>(p, n_wg, stream);
}

}  // namespace mi_fa2
