// Rows to 8 bits: each row's largest magnitude over 127 is its scale, its values are whole multiples of
// it.  Three sources: rows as they are, RMS-normalised rows (after the residual's addition), and the
// fp32 activations of a feed-forward block.
//
// The norm needs no second pass.  With inv = rsqrt(mean(r^2) + eps) the normalised row is
// (r w) inv, so its largest magnitude is max|r w| inv, and
//     value = round((r w) inv / (max|r w| inv / 127)) = round(r w * 127 / max|r w|):
// one reduction brings sum(r^2) and max|r w| together, and inv only enters the scale.  Nothing is
// rounded to 16 bits on the way from r to the value: a value next to a border between two whole
// numbers would change by a whole step (a hundredth of the row's largest) for it.
#include "q8.h"

#include <algorithm>

namespace mi_fa2 {

namespace {

template <typename E>
__device__ __forceinline__ float q8_f(uint16_t x) { return E::lo(x); }
template <typename E>
__device__ __forceinline__ uint16_t q8_r(float x) { return (uint16_t)(E::pack2(x, 0.f) & 0xffffu); }

// Elements 8c .. 8c + 7 of a row of n 16-bit values, zeros past its end.
template <typename E, bool WIDE>
__device__ __forceinline__ void load8(const uint16_t* row, int c, int n, float (&v)[8]) {
  if (WIDE) {   // n is a multiple of 8
    const u32x4 a = 8 * c < n ? ld16(row + 8 * c) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = E::lo(a[e]);
      v[2 * e + 1] = E::hi(a[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 8 * c + e < n ? q8_f<E>(row[8 * c + e]) : 0.f;
  }
}

}  // namespace

// T threads take a row, PER chunks of 8 elements each in registers; PER = 0: any length, the row is
// read twice.
template <typename E, int SRC, bool WIDE, int T, int PER>
__global__ __launch_bounds__(T < 256 ? 256 : T) void q8_quant_kernel(const Q8QuantParams p) {
  constexpr int kRows = T < 256 ? 256 / T : 1;
  // Work-group b runs on XCD b % 8.  Where there are many, all of a panel's rows go to one, whose L2
  // then joins their 16-byte pieces into whole lines.
  constexpr int kPer = 16 / kRows;   // work-groups a panel
  int at = blockIdx.x;
  if (p.spread) {
    const int i = at >> 3;
    at = ((i / kPer) * 8 + (at & 7)) * kPer + i % kPer;
  }
  const int tid = threadIdx.x % T;
  const int row = at * kRows + threadIdx.x / T;
  if (row >= p.M) return;   // (T = 64: whole waves, and no barrier below)
  const int chunks = p.np / 8;
  const uint16_t* x = static_cast<const uint16_t*>(p.x) + (int64_t)row * p.x_st;
  const float* xf = static_cast<const float*>(p.x) + (int64_t)row * p.x_st;
  const uint16_t* y = SRC == kQ8Norm && p.y ? p.y + (int64_t)row * p.y_st : nullptr;
  uint16_t* r_out = SRC == kQ8Norm && p.y ? p.r_out + (int64_t)row * p.r_st : nullptr;

  float ss = 0.f;
  uint32_t top = 0;
  // chunk c of what is held in 8 bits (the norm's factor apart); `first`: counted, and r written
  const auto load = [&](int c, float (&v)[8], bool first) {
    if constexpr (SRC == kQ8Float) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // the rows are padded to whole chunks
        const f32x4 a = 8 * c < p.n ? *reinterpret_cast<const f32x4*>(xf + 8 * c + 4 * h)
                                    : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * h + e] = 8 * c + 4 * h + e < p.n ? a[e] : 0.f;
      }
    } else {
      load8<E, WIDE>(x, c, p.n, v);
      if constexpr (SRC == kQ8Norm) {
        if (y) {
          if (first) {
            float b[8];
            load8<E, WIDE>(y, c, p.n, b);
            u32x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[e] = E::pack2(v[2 * e] + b[2 * e], v[2 * e + 1] + b[2 * e + 1]);
              v[2 * e] = E::lo(o[e]);
              v[2 * e + 1] = E::hi(o[e]);
            }
            if (WIDE) {
              if (8 * c < p.n) *reinterpret_cast<u32x4*>(r_out + 8 * c) = o;
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (8 * c + e < p.n) r_out[8 * c + e] = (uint16_t)(o[e / 2] >> (16 * (e & 1)));
            }
          } else {
            load8<E, WIDE>(r_out, c, p.n, v);   // (this thread's own stores)
          }
        }
        float w[8];
        load8<E, WIDE>(p.norm_w, c, p.n, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (first) ss = __builtin_fmaf(v[e], v[e], ss);
          v[e] *= w[e];
        }
      }
    }
    if (first)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  };

  float kept[PER ? PER : 1][8];
  if constexpr (PER > 0) {
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (tid + k * T < chunks) load(tid + k * T, kept[k], true);
  } else {
    for (int c = tid; c < chunks; c += T) load(c, kept[0], true);
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    if (SRC == kQ8Norm) ss += __shfl_xor(ss, d);
    top = max(top, (uint32_t)__shfl_xor((int)top, d));
  }
  if constexpr (T > 64) {
    __shared__ float part_s[T / 64];
    __shared__ uint32_t part_t[T / 64];
    if ((tid & 63) == 0) {
      part_s[tid >> 6] = ss;
      part_t[tid >> 6] = top;
    }
    __syncthreads();
    ss = 0.f;
    for (int u = 0; u < T / 64; ++u) {
      ss += part_s[u];
      top = max(top, part_t[u]);
    }
  }
  const Q8Factor f = q8_factor(top);
  if (tid == 0)
    p.scale[row] = q8_scale(f, SRC == kQ8Norm ? rsqrtf(ss / (float)p.n + p.eps) : 1.f);
  const auto store = [&](int c, const float (&v)[8]) {
    const u32x2 o = {q8_pack4(v[0], v[1], v[2], v[3], f), q8_pack4(v[4], v[5], v[6], v[7], f)};
    *reinterpret_cast<u32x2*>(p.q + q8_at(row, c, p.np)) = o;
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (tid + k * T < chunks) store(tid + k * T, kept[k]);
  } else {
    for (int c = tid; c < chunks; c += T) {
      load(c, kept[0], false);
      store(c, kept[0]);
    }
  }
}

namespace {

template <typename E, int SRC, bool WIDE>
hipError_t launch_quant_t(Q8QuantParams p, hipStream_t stream) {
  p.spread = p.M > 128;
  // (in whole rounds of the 8 XCDs' panels)
  const int rows = p.spread ? (p.M + 127) / 128 * 128 : p.M;
  if (p.np <= 64 * 4 * 8)
    hipLaunchKernelGGL((q8_quant_kernel<E, SRC, WIDE, 64, 4>), dim3((rows + 3) / 4), dim3(256), 0, stream, p);
  else if (p.np <= 256 * 8 * 8)
    hipLaunchKernelGGL((q8_quant_kernel<E, SRC, WIDE, 256, 8>), dim3(rows), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((q8_quant_kernel<E, SRC, WIDE, 1024, 0>), dim3(rows), dim3(1024), 0, stream, p);
  return hipGetLastError();
}

template <typename E>
hipError_t launch_quant_e(const Q8QuantParams& p, int source, hipStream_t stream) {
  if (source == kQ8Norm)
    return p.wide ? launch_quant_t<E, kQ8Norm, true>(p, stream) : launch_quant_t<E, kQ8Norm, false>(p, stream);
  return p.wide ? launch_quant_t<E, kQ8Plain, true>(p, stream) : launch_quant_t<E, kQ8Plain, false>(p, stream);
}

}  // namespace

hipError_t launch_q8_quant(const Q8QuantParams& p, int dtype, int source, hipStream_t stream) {
  if (source == kQ8Float) return launch_quant_t<BF16, kQ8Float, true>(p, stream);
  return dtype == 0 ? launch_quant_e<BF16>(p, source, stream) : launch_quant_e<FP16>(p, source, stream);
}

// A thread takes 8 values.
template <typename E>
__global__ __launch_bounds__(256) void q8_dequant_kernel(const Q8DequantParams p) {
  const int per_row = (p.n + 7) / 8;
  const int64_t total = (int64_t)p.M * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int row = (int)(i / per_row), c = (int)(i - (int64_t)row * per_row);
    const u32x2 a = *reinterpret_cast<const u32x2*>(p.q + q8_at(row, c, p.np));
    const float s = p.scale[row];
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)(a[e / 4] >> (8 * (e & 3))) * s;
    uint16_t* out = p.out + (int64_t)row * p.out_st + 8 * c;
    if (p.wide) {
      *reinterpret_cast<u32x4*>(out) = u32x4{E::pack2(v[0], v[1]), E::pack2(v[2], v[3]),
                                             E::pack2(v[4], v[5]), E::pack2(v[6], v[7])};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * c + e < p.n) out[e] = q8_r<E>(v[e]);
    }
  }
}

namespace {
// Work-groups of 256 threads for that many pieces, a few each where there are very many.
uint32_t grid_of(int64_t pieces) { return (uint32_t)std::min<int64_t>((pieces + 255) / 256, 1 << 20); }
}  // namespace

hipError_t launch_q8_dequant(const Q8DequantParams& p, int dtype, hipStream_t stream) {
  const int64_t n = (int64_t)p.M * ((p.n + 7) / 8);
  const dim3 grid(grid_of(n));
  if (dtype == 0)
    hipLaunchKernelGGL((q8_dequant_kernel<BF16>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((q8_dequant_kernel<FP16>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

// A weight in panels; a thread moves 16 bytes.
__global__ __launch_bounds__(256) void q8_pack_kernel(const Q8PackParams p) {
  const int per_panel = p.Kp;   // pieces of a panel: 16 Kp / 16
  const int64_t total = (int64_t)p.panels * per_panel;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int panel = (int)(i / per_panel), at = (int)(i - (int64_t)panel * per_panel);
    const int n = at & 15, k = (at >> 6) * 64 + ((at >> 4) & 3) * 16;
    int row = 16 * panel + n;
    bool live = row < p.N;
    if (p.gated) {
      const int f = 8 * panel + (n & 7);
      live = f < p.N / 2;
      row = n < 8 ? f : p.N / 2 + f;
    }
    u32x4 o = {0, 0, 0, 0};
    if (live) {
      const int8_t* src = p.values + (int64_t)row * p.st + k;
      if (p.wide && k + 16 <= p.K) {
        o = *reinterpret_cast<const u32x4*>(src);
      } else {
        for (int e = 0; e < 16; ++e)
          if (k + e < p.K) o[e >> 2] |= (uint32_t)(uint8_t)src[e] << (8 * (e & 3));
      }
    }
    *reinterpret_cast<u32x4*>(p.packed + 16 * i) = o;
  }
}

hipError_t launch_q8_pack(const Q8PackParams& p, hipStream_t stream) {
  const int64_t n = (int64_t)p.panels * p.Kp;
  hipLaunchKernelGGL(q8_pack_kernel, dim3(grid_of(n)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mi_fa2
