// Products of few rows in 8 bits with a packed 8-bit weight: out[M][N] = x[M][K] W[N][K]^T for the tokens
// of a decode step, with the rows' norm and their way to 8 bits in the same launch.
//
// At these sizes a product is one pass over its weight, so the kernel is built to keep as much of W in
// flight as the chip can hold:
//   * A tile is NP panels of W (16 rows each).  A work-group's 8 waves split K; W goes from memory
//     straight into v_mfma_i32_16x16x64_i8 as its A operand, a kilobyte in one run each load, and the
//     next tile's load goes out as soon as this one's has been used.  x is the B operand, 16 tokens per
//     MFMA, MT of them.
//   * For K <= 2048 (KEEP) a wave's share of x stays in registers for all tiles; behind that x is read
//     along with W.
//   * Sums are whole numbers in 32 bits.  The waves' meet in LDS and are added by one wave, another
//     from tile to tile, while the others go on.
//   * Loads go through buffer resources: tokens past M, steps past a wave's share and tiles past a
//     work-group's read as zeros, with no branch around the loads.
// Rows that are not in 8 bits yet (SRC) are brought there first, two by each wave, and pass through LDS into
// the operands' order, while the first weights are on their way.
//
// Bound by the weight stream and a launch's fixed cost.  Measured (bf16, launches in a graph, weights in the
// last-level cache; one token and 16): 2048 x 1536 with norm 3.5 and 4.8 us, rows in 8 bits already 2.5;
// 17920 x 1536 7.0 and 8.8, 6.8 (4.1 TB/s); 151936 x 1536 41.6 and 45.6, 39.5 (5.9 TB/s; a large copy moves
// 5.2).  Weights from memory: 17920 x 1536 8.3 and 9.5.  The norm of 16 rows costs 1.9 to 2.3 us here, where every
// work-group does it over; a launch of its own costs 3.1.
// Two tiles in flight one behind the other in a work-group, a panel each, gained nothing (17920 x 1536 by one token 7.3
// -> 8.0 us); two panels side by side and a second work-group on the CU do (q8_rule.h: 9.0 -> 7.4).
// The tile kernel at the end of the file is for the sizes q8_rule.h says.
#include "q8.h"

#include <algorithm>
#include <type_traits>

namespace mi_fa2 {

namespace {

constexpr int kQrWaves = 8, kQrThreads = 64 * kQrWaves;
constexpr int kQrNone = 0x7ffffff0;   // a byte offset past every resource: reads zeros

// The sums s of four rows of W with token m, whose scale is xs, on their way out: features f .. f + 3
// (GATED: the gate's in lane groups g = 0, 1, the up rows' in 2, 3).  All lanes of the wave call it.
template <typename E, bool GATED>
__device__ __forceinline__ void finish(const Q8Params& p, int f, int m, int g, bool live, float xs, i32x4 s) {
  live = live && m < p.M;
  float v[4];
  if constexpr (GATED) {
    float up[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float ws = f + r < p.N ? p.w_scale[(g < 2 ? 0 : p.N) + f + r] : 0.f;
      v[r] = q8_scaled(s[r], xs, ws);
      up[r] = __shfl_xor(v[r], 32);
    }
    if (g >= 2 || !live || f >= p.N) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = q8_silu_mul(v[r], up[r]);
    // (the rows are padded to whole groups)
    *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + (int64_t)m * p.out_st + f) =
        f32x4{v[0], v[1], v[2], v[3]};
  } else {
    if (!live || f >= p.N) return;
    const uint16_t* res = p.res ? p.res + (int64_t)m * p.res_st + f : nullptr;
    uint16_t* out = static_cast<uint16_t*>(p.out) + (int64_t)m * p.out_st + f;
    if (f + 4 <= p.N) {
      const f32x4 ws = *reinterpret_cast<const f32x4_4*>(p.w_scale + f);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = q8_scaled(s[r], xs, ws[r]);
      if (p.bias) add4<E>(v, *reinterpret_cast<const u32x2_2*>(p.bias + f));
      if (res) add4<E>(v, *reinterpret_cast<const u32x2_2*>(res));
      *reinterpret_cast<u32x2_2*>(out) = u32x2{E::pack2(v[0], v[1]), E::pack2(v[2], v[3])};
      return;
    }
    for (int r = 0; r < p.N - f; ++r) {
      float o = q8_scaled(s[r], xs, p.w_scale[f + r]);
      if (p.bias) o = q8_plus(o, E::lo(p.bias[f + r]));
      if (res) o = q8_plus(o, E::lo(res[r]));
      out[r] = (uint16_t)(E::pack2(o, 0.f) & 0xffffu);
    }
  }
}

// A value rounded to the tensor type.
template <typename E>
__device__ __forceinline__ float rounded(float x) { return E::lo(E::pack2(x, 0.f) & 0xffffu); }
__device__ __forceinline__ float times(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// The sums of a rotation tile (kQrPairs) with token m: dims d .. d + 3 of a head, the lower halves of the
// pairs in lane groups g = 0, 1, the upper in 2, 3.  The projection is rounded, rotated (rounded where the
// model's separate tensor operations round: model.py:58-65) and goes to q or to the token's cache slot.
template <typename E>
__device__ __forceinline__ void finish_rope(const Q8Params& p, int tile, int m, int g, float xs, i32x4 s) {
  const int head = tile >> 3, d = 8 * (tile & 7) + 4 * (g & 1) + 64 * (g >> 1), f = head * kHeadDim + d;
  const f32x4 ws = *reinterpret_cast<const f32x4_4*>(p.w_scale + f);
  float o[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) o[r] = q8_scaled(s[r], xs, ws[r]);
  if (p.bias) add4<E>(o, *reinterpret_cast<const u32x2_2*>(p.bias + f));
#pragma unroll
  for (int r = 0; r < 4; ++r) o[r] = rounded<E>(o[r]);
  const bool live = m < p.M;
  if (head < p.Hq + p.Hkv) {
    const int64_t at = (int64_t)(live ? m : 0) * p.cs_st + d;
    const u32x2 cv = *reinterpret_cast<const u32x2_2*>(p.cos + at), sv = *reinterpret_cast<const u32x2_2*>(p.sin + at);
    float other[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) other[r] = __shfl_xor(o[r], 32);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      // d < 64: x[d] cos[d] - x[d + 64] sin[d];  d >= 64: x[d] cos[d] + x[d - 64] sin[d]
      const float c = r & 1 ? E::hi(cv[r / 2]) : E::lo(cv[r / 2]), n = r & 1 ? E::hi(sv[r / 2]) : E::lo(sv[r / 2]);
      o[r] = q8_plus(rounded<E>(times(o[r], c)), rounded<E>(times(g < 2 ? -other[r] : other[r], n)));
    }
  }
  if (!live) return;
  uint16_t* dst;
  if (head < p.Hq) {
    dst = static_cast<uint16_t*>(p.out) + (int64_t)m * p.out_st + f;
  } else {
    const int slot = p.slots[m];
    if ((unsigned)slot >= (unsigned)p.num_slots) return;   // padding row
    const int h = head - p.Hq;
    dst = (h < p.Hkv ? p.k_pool + h * p.pool_sh : p.v_pool + (h - p.Hkv) * p.pool_sh) + slot * p.pool_st + d;
  }
  *reinterpret_cast<u32x2_2*>(dst) = u32x2{E::pack2(o[0], o[1]), E::pack2(o[2], o[3])};
}

// What a tile's 16 rows of W are: panels; half a panel, whose rows fill the operand twice; the 8 + 8 rows of 8
// rotation pairs of a head of 128.
enum RowsTile { kQrPanels, kQrHalf, kQrPairs };

}  // namespace

// SRC: kQ8Plain, kQ8Norm: x is 16-bit rows; kQ8Float: fp32 rows, 4 at most; kQ8Rows: rows in 8 bits.  NS:
// steps of K (64) a wave takes at a time.
// FT: of fp32 rows, their most.
template <typename E, int MT, int NP, int NS, bool GATED, int SRC, bool KEEP, RowsTile TILE, int FT = 0>
__global__ __launch_bounds__(kQrThreads, 2) void q8_rows_kernel(const Q8Params p) {
  static_assert(SRC == kQ8Rows || MT == 1, "rows come to 8 bits 16 at a time");
  static_assert(KEEP || SRC == kQ8Rows || SRC == kQ8Float, "");
  static_assert(TILE == kQrPanels || (NP == 1 && !GATED), "");
  constexpr int U = NP * MT;
  __shared__ i32x4 red[2][kQrWaves][U][64];
  __shared__ float row_scale[16 * MT];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;

  const int steps = p.Kp >> 6;
  const int lo = wave * steps / kQrWaves, hi = (wave + 1) * steps / kQrWaves;
  const int chunks = KEEP ? 1 : max(1, (hi - lo + NS - 1) / NS);
  const int tiles = TILE == kQrHalf ? 2 * p.panels : (p.panels + NP - 1) / NP;

  // Step i of chunk c of tile t, panel u.
  const auto load_w = [&](int t, int c, int u, int i) -> i32x4 {
    const int s = lo + c * NS + i;
    // (rotation pairs: rows 8 (t % 8) .. + 7 of the head's 128, and those 64, four panels, on)
    const int panel = TILE == kQrHalf ? t >> 1 : TILE == kQrPairs ? (t >> 3) * 8 + ((t & 7) >> 1) : t * NP + u;
    const bool live = TILE == kQrPairs ? t < tiles : panel < p.panels;
    constexpr int kPanels = TILE == kQrPairs ? 5 : 1;
    const __amdgpu_buffer_rsrc_t r =
        make_rsrc(p.w + (int64_t)(live ? panel : 0) * 16 * p.Kp, live ? kPanels * 16 * p.Kp : 0);
    const int at = (TILE == kQrPanels ? lane * 16 : g * 256 + (8 * (t & 1) + (n & 7)) * 16) +
                   (TILE == kQrPairs && n >= 8 ? 64 * p.Kp : 0);
    return __builtin_bit_cast(i32x4, ld16_buf(r, s < hi ? s * 1024 + at : kQrNone));
  };
  // Rows in 8 bits: 16 tokens a panel.
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(p.x, SRC == kQ8Rows ? (p.M + 15) / 16 * 16 * p.Kp : 0);
  // Rows brought to 8 bits here, in LDS: a token's 16 bytes beside those of the others.  The gap keeps a
  // row's pieces off one bank.
  constexpr int kTokens = SRC == kQ8Float ? FT : 16, kPiece = kTokens * 16 + 16;
  constexpr int kMostK = SRC == kQ8Float ? kQ8FloatK : NS * 64 * kQrWaves;
  __shared__ __attribute__((aligned(16))) char pieces[SRC == kQ8Rows ? 16 : kMostK / 16 * kPiece];
  const auto load_x = [&](int c, int j, int i) -> i32x4 {
    const int s = lo + c * NS + i;
    if constexpr (SRC == kQ8Rows)
      return __builtin_bit_cast(i32x4, ld16_buf(xr, s < hi ? j * 16 * p.Kp + s * 1024 + lane * 16 : kQrNone));
    else   // (steps past the share meet weights that are zeros, tokens past the last their own column)
      return *reinterpret_cast<const i32x4*>(pieces + (min(s, steps - 1) * 4 + g) * kPiece + n % kTokens * 16);
  };

  i32x4 x[NS][MT], w[NP][NS];
  const auto first_w = [&] {
#pragma unroll
    for (int u = 0; u < NP; ++u)
#pragma unroll
      for (int i = 0; i < NS; ++i) w[u][i] = load_w(blockIdx.x, 0, u, i);
  };
  if constexpr (SRC == kQ8Rows) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) x[i][j] = load_x(0, j, i);
    first_w();
    if (tid < 16 * MT) row_scale[tid] = tid < p.M ? p.x_scale[tid] : 0.f;
  } else if constexpr (SRC == kQ8Float) {
    // All waves share each row.
    constexpr int kPer = kQ8FloatK / 8 / kQrThreads;   // chunks of 8 a thread
    __shared__ uint32_t part[kQrWaves][kTokens];
    f32x4 v[kTokens][kPer][2];
#pragma unroll
    for (int m = 0; m < kTokens; ++m) {
      const __amdgpu_buffer_rsrc_t rr = make_rsrc(static_cast<const float*>(p.x) + (int64_t)m * p.x_st,
                                                  m < p.M ? p.K * 4 : 0);
#pragma unroll
      for (int k = 0; k < kPer; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          v[m][k][h] = __builtin_bit_cast(f32x4, ld16_buf(rr, (tid + k * kQrThreads) * 32 + h * 16));
    }
    first_w();
    uint32_t top[kTokens];
#pragma unroll
    for (int m = 0; m < kTokens; ++m) {
      top[m] = 0;
#pragma unroll
      for (int k = 0; k < kPer; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) top[m] = max(top[m], __float_as_uint(v[m][k][e / 4][e % 4]) & 0x7fffffffu);
      top[m] = wave_max(top[m]);
      if (lane == 0) part[wave][m] = top[m];
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < kTokens; ++m) {
#pragma unroll
      for (int u = 0; u < kQrWaves; ++u) top[m] = max(top[m], part[u][m]);
      const Q8Factor f = q8_factor(top[m]);
      if (tid == m) row_scale[m] = q8_scale(f, 1.f);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int c = tid + k * kQrThreads;
        if (8 * c < p.Kp)
          *reinterpret_cast<u32x2*>(pieces + (c >> 1) * kPiece + m * 16 + (c & 1) * 8) =
              u32x2{q8_pack4<SRC != kQ8Float>(v[m][k][0][0], v[m][k][0][1], v[m][k][0][2], v[m][k][0][3], f),
                    q8_pack4<SRC != kQ8Float>(v[m][k][1][0], v[m][k][1][1], v[m][k][1][2], v[m][k][1][3], f)};
      }
    }
    __syncthreads();
  } else {
    // Each wave brings rows `wave` and `wave` + 8 there.
    constexpr int kChunks = NS;   // of 8 elements, a lane's share of a row of NS * 512
    u32x4 raw[2][kChunks], nw[kChunks];
    const uint16_t* x16 = static_cast<const uint16_t*>(p.x);
    // (with more than 8 rows, rows past the last: the last again, and not kept)
    if (wave < p.M)
#pragma unroll
      for (int k = 0; k < kChunks; ++k) raw[0][k] = q8_load8(x16 + wave * p.x_st, lane + 64 * k, p.K);
    if (p.M > 8)
#pragma unroll
      for (int k = 0; k < kChunks; ++k)
        raw[1][k] = q8_load8(x16 + min(wave + 8, p.M - 1) * p.x_st, lane + 64 * k, p.K);
    if constexpr (SRC == kQ8Norm)
#pragma unroll
      for (int k = 0; k < kChunks; ++k) nw[k] = q8_load8(p.norm_w, lane + 64 * k, p.K);
    first_w();
    const auto bring = [&](auto rows) {
      constexpr int R = decltype(rows)::value;
      if (p.K != kChunks * 512)
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
#pragma unroll
          for (int h = 0; h < R; ++h) raw[h][k] = q8_cut8(raw[h][k], lane + 64 * k, p.K);
          if constexpr (SRC == kQ8Norm) nw[k] = q8_cut8(nw[k], lane + 64 * k, p.K);
        }
      float v[R][kChunks][8], ss[R];
      uint32_t top[R];
#pragma unroll
      for (int h = 0; h < R; ++h) {
        ss[h] = 0.f;
        top[h] = 0;
#pragma unroll
        for (int k = 0; k < kChunks; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float a = e & 1 ? E::hi(raw[h][k][e / 2]) : E::lo(raw[h][k][e / 2]);
            if constexpr (SRC == kQ8Norm) {
              ss[h] = __builtin_fmaf(a, a, ss[h]);
              a *= e & 1 ? E::hi(nw[k][e / 2]) : E::lo(nw[k][e / 2]);
            }
            v[h][k][e] = a;
            top[h] = max(top[h], __float_as_uint(a) & 0x7fffffffu);
          }
      }
#pragma unroll
      for (int h = 0; h < R; ++h) {
        if (SRC == kQ8Norm) ss[h] = wave_sum(ss[h]);
        top[h] = wave_max(top[h]);
      }
#pragma unroll
      for (int h = 0; h < R; ++h) {
        const int m = wave + 8 * h;
        const Q8Factor f = q8_factor(top[h]);
        if (lane == 0) row_scale[m] = q8_scale(f, SRC == kQ8Norm ? rsqrtf(ss[h] / (float)p.K + p.eps) : 1.f);
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
          const int c = lane + 64 * k;
          if (8 * c < p.Kp)
            *reinterpret_cast<u32x2*>(pieces + (c >> 1) * kPiece + m * 16 + (c & 1) * 8) =
                u32x2{q8_pack4<SRC != kQ8Float>(v[h][k][0], v[h][k][1], v[h][k][2], v[h][k][3], f),
                      q8_pack4<SRC != kQ8Float>(v[h][k][4], v[h][k][5], v[h][k][6], v[h][k][7], f)};
        }
      }
    };
    if (p.M > 8) bring(std::integral_constant<int, 2>{});
    else if (wave < p.M) bring(std::integral_constant<int, 1>{});
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NS; ++i) x[i][0] = load_x(0, 0, i);
  }

  int it = 0;
  for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++it) {
    i32x4 acc[NP][MT];
#pragma unroll
    for (int u = 0; u < NP; ++u)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[u][j] = i32x4{0, 0, 0, 0};
    for (int c = 0; c < chunks; ++c) {
      const bool more = c + 1 < chunks;
      const int nt = more ? t : t + gridDim.x, nc = more ? c + 1 : 0;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        if constexpr (SRC == kQ8Float) x[i][0] = load_x(c, 0, i);
#pragma unroll
        for (int u = 0; u < NP; ++u) {
#pragma unroll
          for (int j = 0; j < MT; ++j)
            acc[u][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][i], x[i][j], acc[u][j], 0, 0, 0);
          w[u][i] = load_w(nt, nc, u, i);
        }
        if constexpr (SRC == kQ8Rows && !KEEP)
#pragma unroll
          for (int j = 0; j < MT; ++j) x[i][j] = load_x(nc, j, i);
      }
    }
    // The waves' sums: lane (n, g) holds rows 4g .. 4g + 3 of a panel for token 16 j + n.  One barrier
    // per tile: the other buffer's readers are past it when they meet this one.
#pragma unroll
    for (int u = 0; u < NP; ++u)
#pragma unroll
      for (int j = 0; j < MT; ++j) red[it & 1][wave][u * MT + j][lane] = acc[u][j];
    __syncthreads();
    for (int u = 0; u < U; ++u) {
      if (((it * U + u) & (kQrWaves - 1)) != wave) continue;
      i32x4 s = red[it & 1][0][u][lane];
#pragma unroll
      for (int v = 1; v < kQrWaves; ++v) s += red[it & 1][v][u][lane];
      const int m = 16 * (u % MT) + n, panel = t * NP + u / MT;
      if constexpr (TILE == kQrPairs) {
        finish_rope<E>(p, t, m, g, row_scale[m], s);
      } else {
        constexpr bool kHalf = TILE == kQrHalf;
        const int f = GATED ? 8 * panel + 4 * (g & 1) : kHalf ? 8 * t + 4 * (g & 1) : 16 * panel + 4 * g;
        finish<E, GATED>(p, f, m, g, !kHalf || g < 2, row_scale[m], s);
      }
    }
  }
}

// A tile of NP panels by 16 MT tokens a work-group, its 8 waves' shares of K each from memory straight into
// the MFMAs, D steps ahead: nothing is shared but the sums, so there is no barrier before the last.  A step is
// (NP + MT) KB for NP MT MFMAs of 16 cycles: bound by the 64 bytes a CU's vector cache gives a cycle, and by
// latency where there are few steps.  64 x 1536 x 8960 9.5-10.0 us (1.4 TB/s of weights), 150 x 896 x 4864 7.1-7.7
// (8 and 10 steps ahead 9.3 and 8.2, and 65 x 512 x 1024 4.2 -> 6.0).
template <typename E, int MT, int NP, int D, bool GATED>
__global__ __launch_bounds__(kQrThreads, 2) void q8_tile_kernel(const Q8Params p) {
  constexpr int U = NP * MT;
  __shared__ i32x4 red[kQrWaves][U][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  // work-group b runs on XCD b % 8: an XCD takes a contiguous share of the tiles, all tokens of a few
  // panels
  const int total = gridDim.x, mt = (p.M + 16 * MT - 1) / (16 * MT);
  const int xcd = blockIdx.x & 7, id = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
  const int tn = id / mt, j0 = (id - tn * mt) * MT, panel0 = tn * NP;
  const int steps = p.Kp >> 6;
  const int lo = wave * steps / kQrWaves, hi = (wave + 1) * steps / kQrWaves;
  const __amdgpu_buffer_rsrc_t wr =
      make_rsrc(p.w + (int64_t)panel0 * 16 * p.Kp, min(NP, p.panels - panel0) * 16 * p.Kp);
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(static_cast<const int8_t*>(p.x) + (int64_t)j0 * 16 * p.Kp,
                                              min(MT, (p.M + 15) / 16 - j0) * 16 * p.Kp);
  i32x4 w[D][NP], x[D][MT], acc[NP][MT];
  const auto load = [&](int d, int s) {
    const int at = s < hi ? s * 1024 + lane * 16 : kQrNone;
#pragma unroll
    for (int u = 0; u < NP; ++u)
      w[d][u] = __builtin_bit_cast(i32x4, ld16_buf(wr, s < hi ? at + u * 16 * p.Kp : kQrNone));
#pragma unroll
    for (int j = 0; j < MT; ++j)
      x[d][j] = __builtin_bit_cast(i32x4, ld16_buf(xr, s < hi ? at + j * 16 * p.Kp : kQrNone));
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load(d, lo + d);
#pragma unroll
  for (int u = 0; u < NP; ++u)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[u][j] = i32x4{0, 0, 0, 0};
  for (int s = lo; s < hi; s += D)
#pragma unroll
    for (int d = 0; d < D; ++d) {
#pragma unroll
      for (int u = 0; u < NP; ++u)
#pragma unroll
        for (int j = 0; j < MT; ++j)
          acc[u][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[d][u], x[d][j], acc[u][j], 0, 0, 0);
      load(d, s + d + D);
    }
#pragma unroll
  for (int u = 0; u < NP; ++u)
#pragma unroll
    for (int j = 0; j < MT; ++j) red[wave][u * MT + j][lane] = acc[u][j];
  __syncthreads();
  for (int u = wave; u < U; u += kQrWaves) {
    i32x4 s = red[0][u][lane];
#pragma unroll
    for (int v = 1; v < kQrWaves; ++v) s += red[v][u][lane];
    const int m = (j0 + u % MT) * 16 + n, panel = panel0 + u / MT;
    finish<E, GATED>(p, GATED ? 8 * panel + 4 * (g & 1) : 16 * panel + 4 * g, m, g, true,
                     p.x_scale[min(m, p.M - 1)], s);
  }
}

namespace {

template <typename E, int MT, int NP, bool GATED, int SRC, RowsTile TILE = kQrPanels>
hipError_t launch_rows_k(const Q8Params& p, const Q8RowsChoice& c, hipStream_t stream) {
  const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(c.grid), dim3(kQrThreads), 0, stream, p); };
  if constexpr (SRC == kQ8Float) {
    constexpr int kSteps = TILE == kQrHalf ? 18 : 9;
    if (c.steps != kSteps) return hipErrorInvalidValue;
    if (p.M == 1) go(q8_rows_kernel<E, MT, NP, kSteps, GATED, SRC, false, TILE, 1>);
    else go(q8_rows_kernel<E, MT, NP, kSteps, GATED, SRC, false, TILE, kQ8FloatMax>);
  } else if (!c.keep) {
    constexpr int kSteps = MT == 1 ? 9 : 6;
    if (c.steps != kSteps) return hipErrorInvalidValue;
    // (q8_plan: no more than 32 rows of these)
    if constexpr (SRC == kQ8Rows && MT < 4 && NP != 2) go(q8_rows_kernel<E, MT, NP, kSteps, GATED, SRC, false, TILE>);
    else return hipErrorInvalidValue;
  } else if constexpr (TILE == kQrHalf) {
    return hipErrorInvalidValue;
  } else {
    switch (c.steps) {
      case 2: go(q8_rows_kernel<E, MT, NP, 2, GATED, SRC, true, TILE>); break;
      case 3: go(q8_rows_kernel<E, MT, NP, 3, GATED, SRC, true, TILE>); break;
      case 4:   // (q8_rows_shape: two panels at most)
        if constexpr (NP < 4) {
          go(q8_rows_kernel<E, MT, NP, 4, GATED, SRC, true, TILE>);
          break;
        }
        [[fallthrough]];
      default: return hipErrorInvalidValue;
    }
  }
  return hipGetLastError();
}

template <typename E, bool GATED, int SRC>
hipError_t launch_rows_m(const Q8Params& p, int n_cus, hipStream_t stream) {
  const Q8RowsChoice c = q8_rows_choice(p.M, p.panels, p.Kp, n_cus, static_cast<Q8Source>(SRC), GATED);
  if constexpr (SRC == kQ8Rows) {
    if (c.mt == 4) return launch_rows_k<E, 4, 1, GATED, SRC>(p, c, stream);
    if (c.mt == 2) return launch_rows_k<E, 2, 1, GATED, SRC>(p, c, stream);
  }
  if constexpr (!GATED && (SRC == kQ8Rows || SRC == kQ8Float))
    if (c.half) return launch_rows_k<E, 1, 1, GATED, SRC, kQrHalf>(p, c, stream);
  if constexpr (SRC != kQ8Float) {
    if (c.panels == 4) return launch_rows_k<E, 1, 4, GATED, SRC>(p, c, stream);
    if (c.panels == 2) return launch_rows_k<E, 1, 2, GATED, SRC>(p, c, stream);
  }
  return launch_rows_k<E, 1, 1, GATED, SRC>(p, c, stream);
}

template <typename E, bool GATED>
hipError_t launch_rows_s(const Q8Params& p, int source, int n_cus, hipStream_t stream) {
  if (source == kQ8Plain) return launch_rows_m<E, GATED, kQ8Plain>(p, n_cus, stream);
  if (source == kQ8Norm) return launch_rows_m<E, GATED, kQ8Norm>(p, n_cus, stream);
  if constexpr (!GATED)
    if (source == kQ8Float) return launch_rows_m<E, GATED, kQ8Float>(p, n_cus, stream);
  return launch_rows_m<E, GATED, kQ8Rows>(p, n_cus, stream);
}

}  // namespace

hipError_t launch_q8_qkv_rope(const Q8Params& p, int dtype, int n_cus, hipStream_t stream) {
  Q8RowsChoice c = q8_rows_choice(p.M, p.panels, p.Kp, n_cus, kQ8Norm, false);
  c.grid = std::min(p.panels, n_cus);   // (a tile is a panel here)
  return dtype == 0 ? launch_rows_k<BF16, 1, 1, false, kQ8Norm, kQrPairs>(p, c, stream)
                    : launch_rows_k<FP16, 1, 1, false, kQ8Norm, kQrPairs>(p, c, stream);
}

hipError_t launch_q8_tile(const Q8Params& p, const Q8Plan& plan, int dtype, bool gated, hipStream_t stream) {
  const dim3 grid(plan.tiles), block(kQrThreads);
  const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, p); };
  const auto sized = [&](auto type, auto gate) {
    using E = decltype(type);
    constexpr bool kGated = decltype(gate)::value;
    if (plan.kernel == kQ8Tile32x32) go(q8_tile_kernel<E, 2, 2, 4, kGated>);
    else if (plan.kernel == kQ8Tile32x64) go(q8_tile_kernel<E, 2, 4, 3, kGated>);
    else go(q8_tile_kernel<E, 4, 4, 3, kGated>);
  };
  if (gated) sized(BF16{}, std::true_type{});
  else if (dtype == 0) sized(BF16{}, std::false_type{});
  else sized(FP16{}, std::false_type{});
  return hipGetLastError();
}

hipError_t launch_q8_rows(const Q8Params& p, int dtype, bool gated, int source, int n_cus,
                          hipStream_t stream) {
  if (gated)
    return dtype == 0 ? launch_rows_s<BF16, true>(p, source, n_cus, stream)
                      : launch_rows_s<FP16, true>(p, source, n_cus, stream);
  return dtype == 0 ? launch_rows_s<BF16, false>(p, source, n_cus, stream)
                    : launch_rows_s<FP16, false>(p, source, n_cus, stream);
}

}  // namespace mi_fa2
