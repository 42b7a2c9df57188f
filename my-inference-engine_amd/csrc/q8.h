// Parameters of the 8-bit projections (q8_quant.hip, q8_rows.hip).
//
// Layouts.  Rows in 8 bits: [rows][Kp] int8, Kp = K rounded up to 128, zeros from K on, one fp32 scale
// a row.  Weights in 8 bits: panels of 16 rows, [panel][Kp / 64][4][16 rows][16 bytes]: lane (n, g) of
// a wave reads the 16 bytes of row n, k = 64 s + 16 g .. + 15, the A operand of
// v_mfma_i32_16x16x64_i8, and a wave's load is 1 KB in one run.  Rows past the last are zeros.  A
// plain panel is rows 16 p .. 16 p + 15; a gated one is gate rows 8 p .. + 7 and the up rows of the
// same features.
#pragma once

#include "fa2_common.h"

namespace mi_fa2 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kQ8Pad = 128;
constexpr float kQ8Least = 0x1p-100f;   // a row's largest magnitude counts as at least this
constexpr int kQ8MaxK = 131072;   // 128 * 127 * K stays below 2^31

__host__ __device__ constexpr int q8_pad(int n) { return (n + kQ8Pad - 1) / kQ8Pad * kQ8Pad; }
__host__ __device__ constexpr int q8_panels(int out, bool gated) {
  return gated ? (out / 2 + 7) / 8 : (out + 15) / 16;
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
  int8_t* q;              // [M][np]
  float* scale;           // [M]
  int32_t M, n, np;
  int32_t wide;           // every row and the norm's weight allow 16-byte accesses
};
enum Q8Source { kQ8Plain = 0, kQ8Norm = 1, kQ8Float = 2 };
hipError_t launch_q8_quant(const Q8QuantParams& p, int dtype, int source, hipStream_t stream);

struct Q8DequantParams {
  const int8_t* q;
  const float* scale;
  uint16_t* out;
  int64_t out_st;
  int32_t M, n, np, wide;
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
  const int8_t* x;        // [M][Kp]
  const float* x_scale;   // [M]
  const int8_t* w;        // packed
  const float* w_scale;   // [N] (gated: [2 N], gate first)
  const uint16_t* bias;   // [N] or NULL
  const uint16_t* res;    // [M][res_st] or NULL; may be out
  int64_t res_st;
  void* out;              // [M][out_st] 16-bit; gated: the activation in fp32
  int64_t out_st;
  int32_t M, N, Kp;       // N: out features (gated: of the activation)
  int32_t panels;
  int32_t quads;          // out, residual and bias allow accesses of 4 elements
};
hipError_t launch_q8_rows(const Q8Params& p, int dtype, bool gated, int n_cus, hipStream_t stream);

}  // namespace mi_fa2
