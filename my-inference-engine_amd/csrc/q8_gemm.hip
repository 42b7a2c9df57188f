// Products of many rows in 8 bits with a packed 8-bit weight: out[M][N] = x[M][K] W[N][K]^T.
#include "q8.h"

#include <algorithm>

namespace mi_fa2 {

namespace {

constexpr int kQgThreads = 256, kQgWaves = 4;

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

template <int N>
__device__ __forceinline__ void wait_loads_and_barrier() {
  // (reads of LDS are finished too: what they read is overwritten behind the barrier)
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <typename E>
__device__ __forceinline__ uint16_t round16(float x) { return (uint16_t)(E::pack2(x, 0.f) & 0xffffu); }

}  // namespace

template <typename E, int NP, int TM, int WN, int ST, bool GATED>
__global__ __launch_bounds__(kQgThreads, 2) void q8_gemm_kernel(const Q8Params p) {
  constexpr int WM = kQgWaves / WN;
  constexpr int TI = NP * 16 / WN / 32, TJ = TM / WM / 32;
  constexpr int kStage = NP * 1024 + TM * 64;
  constexpr int LW = NP / kQgWaves, LX = TM / 16 / kQgWaves, kLoads = LW + LX;
  // the tile on its way out: rows of tokens, 16-bit results or fp32 activations (half as many)
  constexpr int kRow = NP * 16 * 2 + 16;
  constexpr int kLds = ST * kStage > TM * kRow ? ST * kStage : TM * kRow;
  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wm = wave / WN;

  // This work-group's tile.  Work-group b runs on XCD b % 8: an XCD takes a contiguous share of the
  // order, 8 tiles of tokens by one of features after another.
  const int total = gridDim.x, mt = (p.M + TM - 1) / TM, nt = (p.panels + NP - 1) / NP;
  const int xcd = blockIdx.x & 7, id = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
  const int split = id % p.splits, tile = id / p.splits;
  const int group = tile / (8 * nt), first = group * 8, gm = min(8, mt - first);
  const int within = tile - group * 8 * nt;
  const int tn = within / gm, m0 = (first + within - tn * gm) * TM, panel0 = tn * NP;
  const int steps = p.Kp >> 6;
  const int lo = (int)((int64_t)split * steps / p.splits), hi = (int)((int64_t)(split + 1) * steps / p.splits);

  // What this wave loads of a stage (64 of K): the kilobytes of LW panels of W and LX of x.
  const uint64_t w_base = uniform_u64((uint64_t)(p.w + (int64_t)panel0 * 16 * p.Kp));
  const uint32_t w_bytes = (uint32_t)(min(NP, p.panels - panel0) * 16 * p.Kp);
  const uint64_t x_base = uniform_u64((uint64_t)(static_cast<const int8_t*>(p.x) + (int64_t)m0 * p.Kp));
  const uint32_t x_bytes = (uint32_t)(min(TM / 16, (p.M - m0 + 15) / 16) * 16 * p.Kp);
  const uint32_t lds0 = lds_addr_of(lds);
  const int off = wave * 16 * p.Kp + lane * 16;
  const auto issue = [&](int s, int buf) {
    const uint32_t at = lds0 + buf * kStage + wave * 1024;
#pragma unroll
    for (int b = 0; b < LW; ++b)
      lds_dma16_at(w_base, w_bytes, at + b * 4096, off + b * 64 * p.Kp, s * 1024);
#pragma unroll
    for (int b = 0; b < LX; ++b)
      lds_dma16_at(x_base, x_bytes, at + NP * 1024 + b * 4096, off + b * 64 * p.Kp, s * 1024);
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

#pragma unroll
  for (int s = 0; s < ST - 1; ++s)
    if (lo + s < hi) issue(lo + s, s);
  int buf = 0, next = ST - 1;
  for (int s = lo; s < hi; ++s) {
    if (hi - s > ST - 2) wait_loads_and_barrier<(ST - 2) * kLoads>();
    else wait_loads_and_barrier<0>();
    if (s + ST - 1 < hi) issue(s + ST - 1, next);
    const char* wb = wp + buf * kStage;
    const char* xb = xp + buf * kStage;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x4 a[TI], b[TJ];
#pragma unroll
      for (int i = 0; i < TI; ++i) a[i] = *reinterpret_cast<const i32x4*>(wb + i * 2048 + h * 512);
#pragma unroll
      for (int j = 0; j < TJ; ++j) b[j] = *reinterpret_cast<const i32x4*>(xb + j * 2048 + h * 512);
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
    }
    buf = buf + 1 == ST ? 0 : buf + 1;
    next = next + 1 == ST ? 0 : next + 1;
  }

  if (p.splits > 1) {
    // The sums of this share of K go to the workspace, each thread's in a run of its own; the last of
    // the tile's work-groups to arrive adds all of them (whole numbers: in any order).  Relaxed
    // agent-scope atomics, each coherent across the XCDs' L2s by itself; the stores are waited for
    // before the arrival is counted.
    constexpr int kQuads = TI * TJ * 4;
    uint64_t* mine = p.part + ((int64_t)(tile * p.splits + split) * kQuads * kQgThreads + tid) * 2;
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
      const i32x16& t = acc[q / 4 / TJ][q / 4 % TJ];
#pragma unroll
      for (int e = 0; e < 2; ++e)
        __hip_atomic_store(mine + q * kQgThreads * 2 + e,
                           ((uint64_t)(uint32_t)t[q % 4 * 4 + 2 * e + 1] << 32) | (uint32_t)t[q % 4 * 4 + 2 * e],
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* last = reinterpret_cast<int*>(lds);
    if (tid == 0)
      *last = __hip_atomic_fetch_add(p.count + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
              (uint32_t)p.splits - 1;
    __syncthreads();
    if (!*last) return;
    for (int s = 0; s < p.splits; ++s) {
      if (s == split) continue;
      const uint64_t* from = p.part + ((int64_t)(tile * p.splits + s) * kQuads * kQgThreads + tid) * 2;
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        i32x16& t = acc[q / 4 / TJ][q / 4 % TJ];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint64_t v = __hip_atomic_load(from + q * kQgThreads * 2 + e, __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_AGENT);
          t[q % 4 * 4 + 2 * e] += (int)(uint32_t)v;
          t[q % 4 * 4 + 2 * e + 1] += (int)(uint32_t)(v >> 32);
        }
      }
    }
  }

  // Results.  Lane l holds token l % 32 of each 32 x 32 block and rows 8 (r / 4) + 4 (l / 32) + r % 4 of W.
  const int n_first = panel0 * 16 + wn * TI * 32 + 4 * kc;   // of block i, quad q: + 32 i + 8 q
  if constexpr (GATED) {
    // quads 0 and 2 are gate rows, 1 and 3 the up rows of the same features
    constexpr int kF = NP * 8;
    const int f_first = wn * TI * 16 + 4 * kc, f0 = panel0 * 8;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int t = wm * TJ * 32 + j * 32 + r32;
      const float xs = p.x_scale[min(m0 + t, p.M - 1)];
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int f = f_first + 16 * i + 8 * h;
          f32x4 o;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = min(f0 + f + r, p.N - 1);
            const float g = (float)acc[i][j][8 * h + r] * xs * p.w_scale[at];
            const float u = (float)acc[i][j][8 * h + 4 + r] * xs * p.w_scale[p.N + at];
            o[r] = g / (1.f + expf(-g)) * u;
          }
          *reinterpret_cast<f32x4*>(lds + t * kRow + f * 4) = o;
        }
    }
    __syncthreads();
    constexpr int kPieces = kF / 4;   // of 16 bytes a row
    for (int e = tid; e < TM * kPieces; e += kQgThreads) {
      const int t = e / kPieces, c = e % kPieces;
      if (m0 + t < p.M && f0 + 4 * c < p.N)
        *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + (int64_t)(m0 + t) * p.out_st + f0 + 4 * c) =
            *reinterpret_cast<const f32x4*>(lds + t * kRow + c * 16);
    }
  } else if (p.wide) {
    constexpr int kPieces = NP * 2;   // of 16 bytes a row
    uint16_t* out = static_cast<uint16_t*>(p.out);
    __syncthreads();
    if (p.res) {
      for (int e = tid; e < TM * kPieces; e += kQgThreads) {
        const int t = e / kPieces, c = e % kPieces, n = panel0 * 16 + 8 * c;
        if (m0 + t < p.M && n < p.N)
          *reinterpret_cast<u32x4*>(lds + t * kRow + c * 16) = ld16(p.res + (int64_t)(m0 + t) * p.res_st + n);
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int t = wm * TJ * 32 + j * 32 + r32;
      const float xs = p.x_scale[min(m0 + t, p.M - 1)];
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n_first + 32 * i + 8 * q;
          u32x2* at = reinterpret_cast<u32x2*>(lds + t * kRow + (n - panel0 * 16) * 2);
          f32x4 v;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = (float)acc[i][j][4 * q + r] * xs * p.w_scale[min(n + r, p.N - 1)];
          if (p.bias) {
            const u32x2 b = *reinterpret_cast<const u32x2*>(p.bias + min(n, p.N - 4));
            v += f32x4{E::lo(b[0]), E::hi(b[0]), E::lo(b[1]), E::hi(b[1])};
          }
          if (p.res) {
            const u32x2 b = *at;
            v += f32x4{E::lo(b[0]), E::hi(b[0]), E::lo(b[1]), E::hi(b[1])};
          }
          *at = u32x2{E::pack2(v[0], v[1]), E::pack2(v[2], v[3])};
        }
    }
    __syncthreads();
    for (int e = tid; e < TM * kPieces; e += kQgThreads) {
      const int t = e / kPieces, c = e % kPieces, n = panel0 * 16 + 8 * c;
      if (m0 + t < p.M && n < p.N)
        *reinterpret_cast<u32x4*>(out + (int64_t)(m0 + t) * p.out_st + n) =
            *reinterpret_cast<const u32x4*>(lds + t * kRow + c * 16);
    }
  } else {
    // rows that 16-byte accesses do not fit: element by element
    uint16_t* out = static_cast<uint16_t*>(p.out);
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int m = m0 + wm * TJ * 32 + j * 32 + r32;
      if (m >= p.M) continue;
      const float xs = p.x_scale[m];
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int n = n_first + 32 * i + 8 * (e / 4) + e % 4;
          if (n >= p.N) continue;
          float v = (float)acc[i][j][e] * xs * p.w_scale[n];
          if (p.bias) v += E::lo(p.bias[n]);
          if (p.res) v += E::lo(p.res[(int64_t)m * p.res_st + n]);
          out[(int64_t)m * p.out_st + n] = round16<E>(v);
        }
    }
  }
}

namespace {

template <typename E, bool GATED>
hipError_t launch_gemm_e(const Q8Params& p, const Q8Plan& plan, hipStream_t stream) {
  const dim3 grid(plan.tiles * plan.splits), block(kQgThreads);
  if (plan.np == 16)
    hipLaunchKernelGGL((q8_gemm_kernel<E, 16, 128, 2, 3, GATED>), grid, block, 0, stream, p);
  else if (plan.np == 8)
    hipLaunchKernelGGL((q8_gemm_kernel<E, 8, 128, 2, 3, GATED>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((q8_gemm_kernel<E, 4, 64, 2, 4, GATED>), grid, block, 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_q8_gemm(const Q8Params& p, const Q8Plan& plan, int dtype, bool gated, hipStream_t stream) {
  if (gated) return launch_gemm_e<BF16, true>(p, plan, stream);
  return dtype == 0 ? launch_gemm_e<BF16, false>(p, plan, stream)
                    : launch_gemm_e<FP16, false>(p, plan, stream);
}

}  // namespace mi_fa2
