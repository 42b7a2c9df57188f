// Parameters of the 8-bit projections (q8_quant.hip, q8_rows.hip, q8_gemm.hip).
//
// Layouts.  Rows of activations and of weights are held alike, in panels of 16 rows, [panel][Kp / 64][4][16
// rows][16 bytes], Kp = K rounded up to 128, zeros from K on: lane (n, g) of a wave reads the 16 bytes of
// row n, k = 64 s + 16 g .. + 15, an operand of v_mfma_i32_16x16x64_i8, and a wave's load is 1 KB in one
// run (rows as they are would have neighbouring lanes 16 rows apart: a product of 64 tokens by 1536 x
// 8960 24.5 us, in panels 10.7).  One fp32 scale a row.  A gated weight's panel is gate rows 8 p .. + 7 and the
// up rows of the same features.  Rows past a weight's last are zeros; those past the last token are
// whatever was there, and only reach results that nobody keeps.
#pragma once

#include "fa2_common.h"
#include "q8_rule.h"

namespace mi_fa2 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4_4 __attribute__((ext_vector_type(4), aligned(4)));      // at any float
typedef uint32_t u32x4_2 __attribute__((ext_vector_type(4), aligned(2)));   // at any 16-bit element
typedef uint32_t u32x2_2 __attribute__((ext_vector_type(2), aligned(2)));

constexpr int kQ8Pad = 128;
constexpr float kQ8Least = 0x1p-100f;   // a row's largest magnitude counts as at least this
constexpr int kQ8MaxK = 131072;   // 128 * 127 * K stays below 2^31

__host__ __device__ constexpr int q8_pad(int n) { return (n + kQ8Pad - 1) / kQ8Pad * kQ8Pad; }
// Byte of row `row`, k = 8 c (c: a chunk of 8).
__host__ __device__ constexpr int64_t q8_at(int64_t row, int c, int np) {
  return (row >> 4) * 16 * np + (int64_t)(c >> 3) * 1024 + ((c >> 1) & 3) * 256 + (row & 15) * 16 + (c & 1) * 8;
}
__host__ __device__ constexpr int q8_panels(int out, bool gated) {
  return gated ? (out / 2 + 7) / 8 : (out + 15) / 16;
}

// Elements 8c .. 8c + 7 of a row of n 16-bit values at any element, two to a word, zeros past its end.  In two steps, so
// that nothing stands between the loads: q8_load8 (chunks past the last whole one read the row's last 8 elements)
// and q8_cut8.
__device__ __forceinline__ u32x4 q8_load8(const uint16_t* row, int c, int n) {
  if (n >= 8) return *reinterpret_cast<const u32x4_2*>(row + (c < n >> 3 ? 8 * c : n - 8));
  u32x4 a = {0, 0, 0, 0};
  if (c == 0)
    for (int e = 0; e < n; ++e) a[e >> 1] |= (uint32_t)row[e] << (16 * (e & 1));
  return a;
}
__device__ __forceinline__ u32x4 q8_cut8(u32x4 a, int c, int n) {
  if (n < 8) return a;
  u32x4 tail = {0, 0, 0, 0};
  if (n & 7) {   // the last n % 8 of the 8 elements, from the first place on
    const int by = 8 - (n & 7);
    tail = by & 4 ? u32x4{a[2], a[3], 0, 0} : a;
    if (by & 2) tail = u32x4{tail[1], tail[2], tail[3], 0};
    if (by & 1)
      tail = u32x4{tail[0] >> 16 | tail[1] << 16, tail[1] >> 16 | tail[2] << 16, tail[2] >> 16 | tail[3] << 16,
                   tail[3] >> 16};
  }
  return c < n >> 3 ? a : c == n >> 3 ? tail : u32x4{0, 0, 0, 0};
}
// The same stored, elements past n left alone.
__device__ __forceinline__ void q8_store8(uint16_t* row, int c, int n, u32x4 v) {
  if (8 * c + 8 <= n) {
    *reinterpret_cast<u32x4_2*>(row + 8 * c) = v;
  } else {
    for (int e = 0; e < 7; ++e)
      if (8 * c + e < n) row[8 * c + e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
  }
}

// A row's way to 8 bits: its largest magnitude as the bits of |v|, whose order as whole numbers is that of
// the magnitudes, with infinity and NaN above all.
struct Q8Factor {
  float most, f, rest;   // 127 / most is f + rest; a row with an infinity or a NaN: 0
  bool bad;
};
__device__ __forceinline__ Q8Factor q8_factor(uint32_t top) {
  Q8Factor r;
  r.bad = top >= 0x7f800000u;
  r.most = fmaxf(__uint_as_float(top), kQ8Least);
  r.f = r.bad ? 0.f : 127.f / r.most;
  r.rest = r.bad ? 0.f : __builtin_fmaf(-r.f, r.most, 127.f) * (r.f * (1.f / 127.f));
  return r;
}
// inv: what every value is multiplied by beside.
__device__ __forceinline__ float q8_scale(const Q8Factor& r, float inv) {
  return r.bad ? __builtin_nanf("") : r.most * inv / 127.f;
}
// Four values, lowest byte first.  v f is rounded to the nearest whole number, ties to even, by the
// addition of 1.5 * 2^23, whose last place is 1: its low byte is the number's (two's complement).  EXACT: for 16-bit
// rows and their products with a norm's weight, which are short numbers and can lie halfway between two whole ones
// (one row in 128 has a largest magnitude that is a multiple of 127; 4 of 89,600 values of a drawn fp16 case); f
// alone, rounded, would send those to either side.
template <bool EXACT>
__device__ __forceinline__ uint32_t q8_whole(float v, const Q8Factor& r) {
#pragma clang fp contract(off)
  constexpr float kMagic = 12582912.f;
  if constexpr (EXACT) {
    const float y = __builtin_fmaf(v, r.f, v * r.rest);
    return __float_as_uint(y + kMagic);
  } else {
    return __float_as_uint(__builtin_fmaf(v, r.f, kMagic));
  }
}
template <bool EXACT>
__device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d, const Q8Factor& r) {
  // v_perm_b32 selects bytes of {second word, first word}: bytes 0 of both, then the halves
  const uint32_t lo = perm_b32(q8_whole<EXACT>(b, r), q8_whole<EXACT>(a, r), 0x0c0c0400u);
  const uint32_t hi = perm_b32(q8_whole<EXACT>(d, r), q8_whole<EXACT>(c, r), 0x0c0c0400u);
  return r.bad ? 0u : lo | hi << 16;
}

// A wave's sum and maximum, by DPP: each row of 16 lanes by shifts, then the rows' last lanes along.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t q8_dpp(uint32_t v) {   // 0 where no lane is read
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true);
}
__device__ __forceinline__ float wave_sum(float v) {
  const auto add = [&](uint32_t o) { v += __uint_as_float(o); };
  add(q8_dpp<0x111, 0xf>(__float_as_uint(v)));   // row_shr:1, 2, 4, 8
  add(q8_dpp<0x112, 0xf>(__float_as_uint(v)));
  add(q8_dpp<0x114, 0xf>(__float_as_uint(v)));
  add(q8_dpp<0x118, 0xf>(__float_as_uint(v)));
  add(q8_dpp<0x142, 0xa>(__float_as_uint(v)));   // row_bcast:15 to rows 1, 3; row_bcast:31 to rows 2, 3
  add(q8_dpp<0x143, 0xc>(__float_as_uint(v)));
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max(v, q8_dpp<0x111, 0xf>(v));
  v = max(v, q8_dpp<0x112, 0xf>(v));
  v = max(v, q8_dpp<0x114, 0xf>(v));
  v = max(v, q8_dpp<0x118, 0xf>(v));
  v = max(v, q8_dpp<0x142, 0xa>(v));
  v = max(v, q8_dpp<0x143, 0xc>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// A sum with its scales, and what is added to that: each rounded by itself, so that every kernel and every
// alignment gives the same number.
__device__ __forceinline__ float q8_scaled(int s, float x_scale, float w_scale) {
#pragma clang fp contract(off)
  return (float)s * x_scale * w_scale;
}
__device__ __forceinline__ float q8_plus(float a, float b) {
#pragma clang fp contract(off)
  return a + b;
}
// silu(g) u.  The exponential and the reciprocal are the hardware's (a step of fp32 each), and the product in front
// costs |g| steps of e, of which silu sees at most e / (1 + e): far below the 2^-9 of a row's largest at which
// 8 bits round.  (expf and a division: a block of 4,001 x 1536 x 8960 254 us, so 243.)
__device__ __forceinline__ float q8_silu_mul(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * g)) * u;
}
template <typename E>
__device__ __forceinline__ void add4(float (&v)[4], u32x2 b) {
  v[0] = q8_plus(v[0], E::lo(b[0]));
  v[1] = q8_plus(v[1], E::hi(b[0]));
  v[2] = q8_plus(v[2], E::lo(b[1]));
  v[3] = q8_plus(v[3], E::hi(b[1]));
}

// Rows to 8 bits, and back.
struct Q8QuantParams {
  const void* x;          // [M][x_st] 16-bit, or fp32
  int64_t x_st;
  const uint16_t* y;      // added first, or NULL
  int64_t y_st;
  const uint16_t* norm_w; // [n], or NULL
  float eps;
  uint16_t* r_out;        // x + y, with y
  int64_t r_st;
  int8_t* q;              // panels of np
  float* scale;           // [M]
  int32_t M, n, np;
  int32_t spread;         // work-groups are dealt so that a panel's rows share an XCD
};
hipError_t launch_q8_quant(const Q8QuantParams& p, int dtype, int source, hipStream_t stream);

struct Q8DequantParams {
  const int8_t* q;
  const float* scale;
  uint16_t* out;
  int64_t out_st;
  int32_t M, n, np;
};
hipError_t launch_q8_dequant(const Q8DequantParams& p, int dtype, hipStream_t stream);

struct Q8PackParams {
  const int8_t* values;
  int64_t st;
  int8_t* packed;
  int32_t N, K, Kp, panels, gated, wide;
};
hipError_t launch_q8_pack(const Q8PackParams& p, hipStream_t stream);

// A product.
struct Q8Params {
  const void* x;          // panels of Kp, or (few rows) [M][x_st] 16-bit rows to be brought to 8 bits
  int64_t x_st;
  const uint16_t* norm_w; // [K]: their norm's weight
  float eps;
  const float* x_scale;   // [M] of rows in 8 bits
  const int8_t* w;        // packed
  const float* w_scale;   // [N] (gated: [2 N], gate first)
  const uint16_t* bias;   // [N] or NULL
  const uint16_t* res;    // [M][res_st] or NULL; may be out
  int64_t res_st;
  void* out;              // [M][out_st] 16-bit; gated: the activation in fp32
  int64_t out_st;
  int32_t M, N, K, Kp;    // N: out features (gated: of the activation)
  int32_t panels;
  // q/k/v with what follows (few rows): rotary tables [M][cs_st], 128 used, each token's cache slot, one
  // layer of the pools; out is the rotated q
  const uint16_t* cos;
  const uint16_t* sin;
  int64_t cs_st;
  const int32_t* slots;
  uint16_t* k_pool;
  uint16_t* v_pool;
  int64_t pool_st, pool_sh;
  int32_t num_slots, Hq, Hkv;
};
hipError_t launch_q8_rows(const Q8Params& p, int dtype, bool gated, int source, int n_cus,
                          hipStream_t stream);
hipError_t launch_q8_qkv_rope(const Q8Params& p, int dtype, int n_cus, hipStream_t stream);
hipError_t launch_q8_tile(const Q8Params& p, const Q8Plan& plan, int dtype, bool gated, hipStream_t stream);
hipError_t launch_q8_gemm(const Q8Params& p, const Q8Plan& plan, int dtype, bool gated, hipStream_t stream);

}  // namespace mi_fa2
