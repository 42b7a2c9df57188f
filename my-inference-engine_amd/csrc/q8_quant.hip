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
//
// Bound by memory: 16,384 rows of 1,536 with their residual 35.6 us (176 MB, 4.9 TB/s; a large copy moves 5.2),
// 4,096 rows without 5.3 us where they lie in the caches, 7.3 out of memory (19 MB, 2.6 TB/s; before a product that
// evicts them 6.1 to 8.3), 4,001 rows of 8,960 in fp32 28 us (6.4 TB/s: out of the last-level cache), one row 2.9 us.
// All of a thread's loads go out before the first is used.
#include "q8.h"

#include <algorithm>

namespace mi_fa2 {

namespace {

template <typename E>
__device__ __forceinline__ void unpack8(u32x4 a, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = E::lo(a[e]);
    v[2 * e + 1] = E::hi(a[e]);
  }
}

}  // namespace

// T threads take a row, PER chunks of 8 elements each in registers; PER = 0: any length, the row is
// read twice.
template <typename E, int SRC, int T, int PER>
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
  // A row is a wave's or a work-group's: its address is uniform.
  const int64_t urow = __builtin_amdgcn_readfirstlane(row);
  const uint16_t* x = static_cast<const uint16_t*>(p.x) + urow * p.x_st;
  const __amdgpu_buffer_rsrc_t xf =
      make_rsrc(static_cast<const float*>(p.x) + urow * p.x_st, SRC == kQ8Float ? p.n * 4 : 0);
  const bool add = SRC == kQ8Norm && p.y;
  const uint16_t* y = add ? p.y + urow * p.y_st : nullptr;
  uint16_t* r = add ? p.r_out + urow * p.r_st : nullptr;

  float ss = 0.f;
  uint32_t top = 0;
  // A chunk as it is loaded, and what of it is held in 8 bits (the norm's factor apart); `first`: counted, and
  // r written.
  struct Chunk {
    u32x4 x[SRC == kQ8Float ? 2 : 1], y, w;
  };
  const auto load = [&](int c, bool first) {
    Chunk k{};
    if constexpr (SRC == kQ8Float) {   // (zeros past the row's end)
#pragma unroll
      for (int h = 0; h < 2; ++h) k.x[h] = ld16_buf(xf, 32 * c + 16 * h);
    } else {
      k.x[0] = q8_load8(add && !first ? r : x, c, p.n);   // (the second time r is this thread's own stores)
      if (add && first) k.y = q8_load8(y, c, p.n);
      if constexpr (SRC == kQ8Norm) k.w = q8_load8(p.norm_w, c, p.n);
    }
    return k;
  };
  const auto cut = [&](int c, Chunk& k) {
    if constexpr (SRC != kQ8Float) {
      k.x[0] = q8_cut8(k.x[0], c, p.n);
      k.y = q8_cut8(k.y, c, p.n);
      k.w = q8_cut8(k.w, c, p.n);
    }
  };
  const auto take = [&](int c, const Chunk& k, float (&v)[8], bool first) {
    if constexpr (SRC == kQ8Float) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(k.x[e / 4][e % 4]);
    } else {
      unpack8<E>(k.x[0], v);
      if constexpr (SRC == kQ8Norm) {
        if (add && first) {
          float b[8];
          unpack8<E>(k.y, b);
          u32x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = E::pack2(v[2 * e] + b[2 * e], v[2 * e + 1] + b[2 * e + 1]);
          unpack8<E>(o, v);
          q8_store8(r, c, p.n, o);
        }
        float w[8];
        unpack8<E>(k.w, w);
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
    Chunk k[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) k[i] = load(tid + i * T, true);
    if (p.n != PER * T * 8)
#pragma unroll
      for (int i = 0; i < PER; ++i) cut(tid + i * T, k[i]);
#pragma unroll
    for (int i = 0; i < PER; ++i) take(tid + i * T, k[i], kept[i], true);
  } else {
    for (int c = tid; c < chunks; c += T) {
      Chunk k = load(c, true);
      cut(c, k);
      take(c, k, kept[0], true);
    }
  }
  if (SRC == kQ8Norm) ss = wave_sum(ss);
  top = wave_max(top);
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
    const u32x2 o = {q8_pack4<SRC != kQ8Float>(v[0], v[1], v[2], v[3], f),
                     q8_pack4<SRC != kQ8Float>(v[4], v[5], v[6], v[7], f)};
    *reinterpret_cast<u32x2*>(p.q + q8_at(row, c, p.np)) = o;
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (tid + k * T < chunks) store(tid + k * T, kept[k]);
  } else {
    for (int c = tid; c < chunks; c += T) {
      Chunk k = load(c, false);
      cut(c, k);
      take(c, k, kept[0], false);
      store(c, kept[0]);
    }
  }
}

namespace {

template <typename E, int SRC, int T, int PER, int LAST>
void launch_quant_per(const Q8QuantParams& p, dim3 grid, hipStream_t stream) {
  if constexpr (PER < LAST)
    if (p.np > T * 8 * PER) return launch_quant_per<E, SRC, T, PER + 1, LAST>(p, grid, stream);
  hipLaunchKernelGGL((q8_quant_kernel<E, SRC, T, PER>), grid, dim3(T < 256 ? 256 : T), 0, stream, p);
}

template <typename E, int SRC>
hipError_t launch_quant_t(Q8QuantParams p, hipStream_t stream) {
  p.spread = p.M > 128;
  // (in whole rounds of the 8 XCDs' panels)
  const int rows = p.spread ? (p.M + 127) / 128 * 128 : p.M;
  // A wave a row where four chunks a lane hold it; else a work-group, a large one where there are few rows (64
  // of 8,960: 3.3 us, of 256 threads 3.8).
  if (p.np <= 64 * 4 * 8) launch_quant_per<E, SRC, 64, 1, 4>(p, dim3((rows + 3) / 4), stream);
  else if (p.M <= 64 && p.np <= 1024 * 8 * 4) launch_quant_per<E, SRC, 1024, 1, 4>(p, dim3(rows), stream);
  else if (p.np <= 256 * 8 * 8) launch_quant_per<E, SRC, 256, 2, 8>(p, dim3(rows), stream);
  else launch_quant_per<E, SRC, 1024, 0, 0>(p, dim3(rows), stream);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_q8_quant(const Q8QuantParams& p, int dtype, int source, hipStream_t stream) {
  if (source == kQ8Float) return launch_quant_t<BF16, kQ8Float>(p, stream);
  if (source == kQ8Norm)
    return dtype == 0 ? launch_quant_t<BF16, kQ8Norm>(p, stream) : launch_quant_t<FP16, kQ8Norm>(p, stream);
  return dtype == 0 ? launch_quant_t<BF16, kQ8Plain>(p, stream) : launch_quant_t<FP16, kQ8Plain>(p, stream);
}

// A thread takes 16 values of one row, a wave 16 rows' 64: it reads 1 KB in one run and writes each row's
// 128 bytes.
template <typename E>
__global__ __launch_bounds__(256) void q8_dequant_kernel(const Q8DequantParams p) {
  const int per_panel = p.np;   // 16-byte pieces
  const int64_t total = (int64_t)((p.M + 15) / 16) * per_panel;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t panel = i / per_panel;
    const int at = (int)(i - panel * per_panel);
    const int64_t row = panel * 16 + (at & 15);
    if (row >= p.M) continue;
    const u32x4 a = *reinterpret_cast<const u32x4*>(p.q + 16 * i);
    const float s = p.scale[row];
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = (float)(int8_t)(a[e / 4] >> (8 * (e & 3))) * s;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      q8_store8(p.out + row * p.out_st, (at >> 4) * 2 + h, p.n,
                u32x4{E::pack2(v[8 * h], v[8 * h + 1]), E::pack2(v[8 * h + 2], v[8 * h + 3]),
                      E::pack2(v[8 * h + 4], v[8 * h + 5]), E::pack2(v[8 * h + 6], v[8 * h + 7])});
  }
}

namespace {
// Work-groups of 256 threads for that many pieces, a few each where there are very many.
uint32_t grid_of(int64_t pieces) { return (uint32_t)std::min<int64_t>((pieces + 255) / 256, 1 << 20); }
}  // namespace

hipError_t launch_q8_dequant(const Q8DequantParams& p, int dtype, hipStream_t stream) {
  const dim3 grid(grid_of((int64_t)((p.M + 15) / 16) * p.np));
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
