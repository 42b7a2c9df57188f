// Products of rows in 8 bits with a packed 8-bit weight: out[M][N] = x[M][K] W[N][K]^T.
//
// A tile is one panel of W (16 rows) by 16 MT tokens; the 8 waves of a work-group split K, and W goes from
// memory straight into v_mfma_i32_16x16x64_i8 as its A operand, x as the B operand.  Sums are whole
// numbers in 32 bits, so their order does not matter.
#include "q8.h"

#include <algorithm>

namespace mi_fa2 {

namespace {
constexpr int kQrWaves = 8, kQrThreads = 64 * kQrWaves;
}

template <typename E, int MT, bool GATED>
__global__ __launch_bounds__(kQrThreads) void q8_rows_kernel(const Q8Params p) {
  __shared__ i32x4 red[kQrWaves][MT][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int panel = blockIdx.x;
  const int m0 = blockIdx.y * 16 * MT;
  const int steps = p.Kp >> 6;
  const int lo = wave * steps / kQrWaves, hi = (wave + 1) * steps / kQrWaves;

  const int8_t* w = p.w + (int64_t)panel * 16 * p.Kp;
  const int rows = min(16 * MT, p.M - m0);
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(w, 16 * p.Kp);
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(p.x + (int64_t)m0 * p.Kp, rows * p.Kp);
  i32x4 acc[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) acc[j] = i32x4{0, 0, 0, 0};
  for (int s = lo; s < hi; ++s) {
    const i32x4 a = __builtin_bit_cast(i32x4, ld16_buf(wr, s * 1024 + lane * 16));
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const i32x4 b = __builtin_bit_cast(i32x4, ld16_buf(xr, (16 * j + n) * p.Kp + s * 64 + g * 16));
      acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc[j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) red[wave][j][lane] = acc[j];
  __syncthreads();
  for (int j = wave; j < MT; j += kQrWaves) {
    i32x4 s = red[0][j][lane];
#pragma unroll
    for (int u = 1; u < kQrWaves; ++u) s += red[u][j][lane];
    const int m = m0 + 16 * j + n;
    const bool live = m < p.M;
    const float xs = p.x_scale[live ? m : m0];
    float v[4];
    if constexpr (GATED) {
      const int f = 8 * panel + 4 * (g & 1);
      float u[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float ws = f + r < p.N ? p.w_scale[(g < 2 ? 0 : p.N) + f + r] : 0.f;
        v[r] = (float)s[r] * xs * ws;
        u[r] = __shfl_xor(v[r], 32);
      }
      if (g >= 2 || !live || f >= p.N) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = v[r] / (1.f + expf(-v[r])) * u[r];
      // (the rows are padded to whole groups)
      *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + (int64_t)m * p.out_st + f) =
          f32x4{v[0], v[1], v[2], v[3]};
    } else {
      const int f = 16 * panel + 4 * g;
      if (!live || f >= p.N) continue;
      const uint16_t* res = p.res ? p.res + (int64_t)m * p.res_st + f : nullptr;
      uint16_t* out = static_cast<uint16_t*>(p.out) + (int64_t)m * p.out_st + f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (f + r >= p.N) break;
        float t = (float)s[r] * xs * p.w_scale[f + r];
        if (p.bias) t += E::lo(p.bias[f + r]);
        if (res) t += E::lo(res[r]);
        out[r] = (uint16_t)(E::pack2(t, 0.f) & 0xffffu);
      }
    }
  }
}

namespace {

template <typename E, bool GATED>
hipError_t launch_rows_e(const Q8Params& p, hipStream_t stream) {
  const int mt = p.M <= 16 ? 1 : p.M <= 32 ? 2 : 4;
  const dim3 grid(p.panels, (p.M + 16 * mt - 1) / (16 * mt));
  if (mt == 1)
    hipLaunchKernelGGL((q8_rows_kernel<E, 1, GATED>), grid, dim3(kQrThreads), 0, stream, p);
  else if (mt == 2)
    hipLaunchKernelGGL((q8_rows_kernel<E, 2, GATED>), grid, dim3(kQrThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((q8_rows_kernel<E, 4, GATED>), grid, dim3(kQrThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_q8_rows(const Q8Params& p, int dtype, bool gated, int n_cus, hipStream_t stream) {
  (void)n_cus;
  if (gated) return launch_rows_e<BF16, true>(p, stream);
  return dtype == 0 ? launch_rows_e<BF16, false>(p, stream) : launch_rows_e<FP16, false>(p, stream);
}

}  // namespace mi_fa2
