// Products of many rows in 8 bits with a packed 8-bit weight: out[M][N] = x[M][K] W[N][K]^T.
//
// A work-group of 4 waves (8) computes TM tokens by NP panels (64 x 64, a wave 32 x 32; 128 x 128, a wave 64 x 64;
// up to 256 x 256, a wave 64 tokens by 128 features) with v_mfma_i32_32x32x32_i8.  W is the A operand, so a lane's
// four sums in a row are four features of one token.  Both operands come in panels (q8.h): a stage of 64 of K is
// NP + TM / 16 loads of 1 KB straight into LDS, and a 32 x 32 operand is read out of two panels' kilobytes, 16 lanes
// in a run, with no two on a bank.  ST stages are in flight.  A stage's operands are read during the MFMAs of the
// stage before, behind one barrier a stage; the loads ST stages ahead follow between the second half of the MFMAs
// (reads, then MFMAs, then loads, without that: 6001 x 6144 x 4096 153-159 us where this took 148-152).
// Results: the tile's scales wait in LDS, loaded with the first stage; the sums are scaled, meet bias and
// residual in fp32, and leave through LDS as whole rows, past the caches (143 -> 121 us for 4001 x 17920 x 1536
// against stores that stay in the L2).  GATED: quads of gate and up rows of the same features lie in one lane,
// silu(g) u leaves in fp32: in bfloat16 the values between half the row's largest and the largest lie half a
// step of the 8 bits apart, so one in eight of them would move by a whole step.
//
// Measured (rows in 8 bits, launches in a graph, several cards): 8192^3 426-459 us (2.40-2.58 POP/s; the library's
// int8 product 2.06), 4096^3 60-61, 6001 x 6144 x 4096 130-137 (the library's 180), 4096 x 17920 x 1536
// 112-122 (140), 4001 x 1536 x 8960 53-59 (70), 4096 x 2048 x 1536 16.1-20.1 (25.0).  What bounds the long ones is
// power: the MFMAs alone run at 3.8 POP/s; with 128 x 128 tiles 8192^3 ran at 1.4 GHz (a stage of three work-groups
// 900 cycles for 768 of MFMAs), and on zeros at 1.9 GHz and 3.1 POP/s.  Larger tiles move fewer bytes for a product
// (128 x 128 483 us, 128 x 256 441, 256 x 256 426).  K of 1536 is only 24 stages: there a tile's start and its
// results show (without the stores 4001 x 17920 x 1536 took 119 us for 121, 4096 x 2048 x 1536 18.2 for 20.1).
#include "q8.h"

#include <algorithm>

namespace mi_fa2 {

namespace {


// lds_dma16 with a wave-uniform byte offset beside the lanes' (which alone are held against `bytes`).
__device__ __forceinline__ void lds_dma16_at(uint64_t base, uint32_t bytes, uint32_t lds_addr,
                                             int voffset, int soffset) {
  const u32x4 rsrc = {(uint32_t)base, (uint32_t)(base >> 32) & 0xffffu, bytes, 0x00020000u};
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, %3 offen lds"
      :
      : "s"(lds_addr), "v"(voffset), "s"(rsrc), "s"(soffset)
      : "memory");
}

// Four bytes a lane, at LDS byte lds_addr + 4 lane.
__device__ __forceinline__ void lds_dma4(uint64_t base, uint32_t bytes, uint32_t lds_addr, int voffset) {
  const u32x4 rsrc = {(uint32_t)base, (uint32_t)(base >> 32) & 0xffffu, bytes, 0x00020000u};
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %1, %2, 0 offen lds"
      :
      : "s"(lds_addr), "v"(voffset), "s"(rsrc)
      : "memory");
}

template <int N>
__device__ __forceinline__ void wait_loads_and_barrier() {
  // (reads of LDS are finished too: what they read is overwritten behind the barrier)
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

}  // namespace

// WN of the waves stand side by side along W.  A CU holds three work-groups of 128 x 128 (135 registers), two of
// the larger tiles, or one of 8 waves (256 x 256: as many waves, a third fewer loads); fewer hide less (6001 x 6144
// x 4096 with 128 x 128 in four stages, and so two a CU, 150 -> 186 us; with 128 x 192 in four, and so one, 137 -> 222).
template <typename E, int NP, int TM, int WN, int ST, bool GATED, int WAVES = 4>
__global__ __launch_bounds__(WAVES * 64, NP * TM > 1024 ? 2 : NP == 8 ? 3 : 4) void q8_gemm_kernel(const Q8Params p) {
  constexpr int kThreads = WAVES * 64, WM = WAVES / WN;
  constexpr int TI = NP * 16 / WN / 32, TJ = TM / WM / 32;
  constexpr int kStage = NP * 1024 + TM * 64;
  constexpr int LW = NP / WAVES, LX = TM / 16 / WAVES, kLoads = LW + LX;
  // the tile on its way out: rows of tokens, 16-bit results or fp32 activations (half as many)
  constexpr int kRow = NP * 16 * 2 + 16;
  constexpr int kTile = ST * kStage > TM * kRow ? ST * kStage : TM * kRow;
  __shared__ __attribute__((aligned(1024))) char lds[kTile + (2 * NP * 16 + TM) * 4];
  float* w_scale = reinterpret_cast<float*>(lds + kTile);   // of the tile's rows of W and tokens
  float* x_scale = w_scale + NP * 16;
  float* bias = x_scale + TM;   // in fp32
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wm = wave / WN;

  // This work-group's tile.  Work-group b runs on XCD b % 8: an XCD takes a contiguous share of the
  // order, 8 tiles of tokens by one of features after another.
  const int total = gridDim.x, mt = (p.M + TM - 1) / TM, nt = (p.panels + NP - 1) / NP;
  const int xcd = blockIdx.x & 7, id = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
  const int group = id / (8 * nt), first = group * 8, gm = min(8, mt - first);
  const int within = id - group * 8 * nt;
  const int tn = within / gm, m0 = (first + within - tn * gm) * TM, panel0 = tn * NP;
  const int steps = p.Kp >> 6;

  // What this wave loads of a stage (64 of K): the kilobytes of LW panels of W and LX of x.
  const uint64_t w_base = uniform_u64((uint64_t)(p.w + (int64_t)panel0 * 16 * p.Kp));
  const uint32_t w_bytes = (uint32_t)(min(NP, p.panels - panel0) * 16 * p.Kp);
  const uint64_t x_base = uniform_u64((uint64_t)(static_cast<const int8_t*>(p.x) + (int64_t)m0 * p.Kp));
  const uint32_t x_bytes = (uint32_t)(min(TM / 16, (p.M - m0 + 15) / 16) * 16 * p.Kp);
  const uint32_t lds0 = lds_addr_of(lds);
  const int off = wave * 16 * p.Kp + lane * 16;
  // the scales, 64 rows or tokens a wave
  if (wave < NP / 4) {
    const int r = panel0 * 16 + wave * 64 + lane, f = (r >> 4) * 8 + (r & 7);
    const int at = GATED ? (f < p.N ? (r & 8 ? p.N : 0) + f : -1) : (r < p.N ? r : -1);
    lds_dma4(uniform_u64((uint64_t)p.w_scale), 0x7fffffffu, lds0 + kTile + wave * 256, at < 0 ? 0 : at * 4);
  }
  if (wave < TM / 64) {
    const int t = min(m0 + wave * 64 + lane, p.M - 1);
    lds_dma4(uniform_u64((uint64_t)p.x_scale), 0x7fffffffu, lds0 + kTile + NP * 64 + wave * 256, t * 4);
  }
  const auto load = [&](int i, int s, int buf) {   // one of a stage's kLoads
    const uint32_t at = lds0 + buf * kStage + wave * 1024;
    if (i < LW) lds_dma16_at(w_base, w_bytes, at + i * WAVES * 1024, off + i * WAVES * 16 * p.Kp, s * 1024);
    else
      lds_dma16_at(x_base, x_bytes, at + (NP + (i - LW) * WAVES) * 1024, off + (i - LW) * WAVES * 16 * p.Kp, s * 1024);
  };

  i32x16 acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  // Operands: lane l holds row (token) l % 32 and the 16 bytes of k 16 (l / 32) .. of each half step.
  const int r32 = lane & 31, kc = lane >> 5;
  const int operand = (r32 >> 4) * 1024 + kc * 256 + (r32 & 15) * 16;
  const char* wp = lds + wn * TI * 2048 + operand;
  const char* xp = lds + NP * 1024 + wm * TJ * 2048 + operand;

  // A stage's operands are read while the MFMAs of the one before run: the reads, then the loads of the
  // stage ST ahead, one or two behind each MFMA.
  constexpr int kReads = 2 * (TI + TJ), kMfmas = 2 * TI * TJ;
  i32x4 a[2][2][TI], b[2][2][TJ];
  const auto read = [&](int set, int i, int buf) {   // one of a stage's kReads
    const int h = i / (TI + TJ), t = i % (TI + TJ);
    if (t < TI) a[set][h][t] = *reinterpret_cast<const i32x4*>(wp + buf * kStage + t * 2048 + h * 512);
    else b[set][h][t - TI] = *reinterpret_cast<const i32x4*>(xp + buf * kStage + (t - TI) * 2048 + h * 512);
  };
#pragma unroll
  for (int s = 0; s < ST; ++s)
    if (s < steps)
#pragma unroll
      for (int i = 0; i < kLoads; ++i) load(i, s, s);
  if (steps >= ST) wait_loads_and_barrier<(ST - 1) * kLoads>();
  else wait_loads_and_barrier<0>();
#pragma unroll
  for (int i = 0; i < kReads; ++i) read(0, i, 0);
  int buf = 0;   // stage s
  const auto stage = [&](int s, int set) {
    const int next = buf + 1 == ST ? 0 : buf + 1;
    // stage s + 1 is there, and stage s has been read by all waves
    if (steps - s >= ST) wait_loads_and_barrier<(ST - 2) * kLoads>();
    else wait_loads_and_barrier<0>();
    const bool more = s + ST < steps;
#pragma unroll
    for (int k = 0; k < kMfmas; ++k) {
      const int h = k / (TI * TJ), i = k % (TI * TJ) / TJ, j = k % TJ;
      acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[set][h][i], b[set][h][j], acc[i][j], 0, 0, 0);
      constexpr int kHalf = kMfmas / 2;
#pragma unroll
      for (int t = 0; t < kReads; ++t)
        if (k == t * kHalf / kReads) read(set ^ 1, t, next);
      if (more)
#pragma unroll
        for (int t = 0; t < kLoads; ++t)
          if (k == kHalf + t * (kMfmas - kHalf) / kLoads) load(t, s + ST, buf);
      __builtin_amdgcn_sched_barrier(0);
    }
    buf = next;
  };
  for (int s = 0; s < steps; s += 2) {
    stage(s, 0);
    if (s + 1 < steps) stage(s + 1, 1);
  }

  // Results.  Lane l holds token l % 32 of each 32 x 32 block and rows 8 (r / 4) + 4 (l / 32) + r % 4 of W.
  const int w_first = wn * TI * 32 + 4 * kc;   // of block i, quad q: + 32 i + 8 q
  if constexpr (GATED) {
    __syncthreads();
    // quads 0 and 2 are gate rows, 1 and 3 the up rows of the same features
    constexpr int kPieces = NP * 2;   // of 16 bytes a row
    const int f0 = panel0 * 8;
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 gs = *reinterpret_cast<const f32x4*>(w_scale + w_first + 32 * i + 16 * h);
        const f32x4 us = *reinterpret_cast<const f32x4*>(w_scale + w_first + 32 * i + 16 * h + 8);
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
          const int t = wm * TJ * 32 + j * 32 + r32;
          const float xs = x_scale[t];
          f32x4 o;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float g = q8_scaled(acc[i][j][8 * h + r], xs, gs[r]);
            const float u = q8_scaled(acc[i][j][8 * h + 4 + r], xs, us[r]);
            o[r] = q8_silu_mul(g, u);
          }
          *reinterpret_cast<f32x4*>(lds + t * kRow + (wn * TI * 16 + 4 * kc + 16 * i + 8 * h) * 4) = o;
        }
      }
    __syncthreads();
    float* out = static_cast<float*>(p.out) + (int64_t)m0 * p.out_st + f0;
#pragma unroll
    for (int e = 0; e < TM * kPieces / kThreads; ++e) {
      const int t = (tid + e * kThreads) / kPieces, c = (tid + e * kThreads) % kPieces;
      if (m0 + t < p.M && f0 + 4 * c < p.N)
        *reinterpret_cast<f32x4*>(out + t * p.out_st + 4 * c) =
            *reinterpret_cast<const f32x4*>(lds + t * kRow + c * 16);
    }
  } else {
    constexpr int kPieces = NP * 2;   // of 16 bytes a row
    uint16_t* out = static_cast<uint16_t*>(p.out) + (int64_t)m0 * p.out_st + panel0 * 16;
    const int n_left = p.N - panel0 * 16;
    uint16_t my_bias = 0;
    if (p.bias && tid < NP * 16 && tid < n_left) my_bias = p.bias[panel0 * 16 + tid];
    if (p.res) {
      // the residual takes its place in LDS, where the sums then meet it
      constexpr int kEach = TM * kPieces / kThreads, kBatch = kEach > 12 ? kEach / 2 : kEach;
#pragma unroll
      for (int first = 0; first < kEach; first += kBatch) {
        u32x4 res[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          const int at = tid + (first + e) * kThreads, m = min(m0 + at / kPieces, p.M - 1);
          res[e] = q8_load8(p.res + m * p.res_st + panel0 * 16, at % kPieces, n_left);
        }
        if (first == 0) __syncthreads();
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          const int at = tid + (first + e) * kThreads, c = at % kPieces;
          *reinterpret_cast<u32x4*>(lds + at / kPieces * kRow + c * 16) = q8_cut8(res[e], c, n_left);
        }
      }
    }
    if (tid < NP * 16) bias[tid] = E::lo(my_bias);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = w_first + 32 * i + 8 * q;
        const f32x4 ws = *reinterpret_cast<const f32x4*>(w_scale + n), bs = *reinterpret_cast<const f32x4*>(bias + n);
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
          const int t = wm * TJ * 32 + j * 32 + r32;
          const float xs = x_scale[t];
          u32x2* at = reinterpret_cast<u32x2*>(lds + t * kRow + n * 2);
          float v[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            v[r] = q8_scaled(acc[i][j][4 * q + r], xs, ws[r]);
            if (p.bias) v[r] = q8_plus(v[r], bs[r]);
          }
          if (p.res) add4<E>(v, *at);
          *at = u32x2{E::pack2(v[0], v[1]), E::pack2(v[2], v[3])};
        }
      }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < TM * kPieces / kThreads; ++e) {
      const int t = (tid + e * kThreads) / kPieces, c = (tid + e * kThreads) % kPieces;
      const u32x4 v = *reinterpret_cast<const u32x4*>(lds + t * kRow + c * 16);
      if (m0 + t >= p.M) break;
      if (8 * c + 8 <= n_left)
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4_2*>(out + t * p.out_st + 8 * c));
      else
        q8_store8(out + t * p.out_st, c, n_left, v);
    }
  }
}

namespace {

template <typename E, bool GATED>
hipError_t launch_gemm_e(const Q8Params& p, const Q8Plan& plan, hipStream_t stream) {
  const auto go = [&](auto kernel, int threads = 256) {
    hipLaunchKernelGGL(kernel, dim3(plan.tiles), dim3(threads), 0, stream, p);
  };
  switch (plan.kernel) {
    case kQ8Gemm64: go(q8_gemm_kernel<E, 4, 64, 2, 4, GATED>); break;
    case kQ8Gemm128: go(q8_gemm_kernel<E, 8, 128, 2, 3, GATED>); break;
    case kQ8Gemm128x192: go(q8_gemm_kernel<E, 12, 128, 2, 3, GATED>); break;
    case kQ8Gemm192x128: go(q8_gemm_kernel<E, 8, 192, 2, 3, GATED>); break;
    case kQ8Gemm128x256: go(q8_gemm_kernel<E, 16, 128, 2, 3, GATED>); break;
    case kQ8Gemm192x192: go(q8_gemm_kernel<E, 12, 192, 2, 3, GATED>); break;
    case kQ8Gemm256x256: go(q8_gemm_kernel<E, 16, 256, 2, 4, GATED, 8>, 512); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_q8_gemm(const Q8Params& p, const Q8Plan& plan, int dtype, bool gated, hipStream_t stream) {
  if (gated) return launch_gemm_e<BF16, true>(p, plan, stream);
  return dtype == 0 ? launch_gemm_e<BF16, false>(p, plan, stream)
                    : launch_gemm_e<FP16, false>(p, plan, stream);
}

}  // namespace mi_fa2
