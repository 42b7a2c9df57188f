/*
 * C ABI of libmi_q8.so: the projections of a decoder layer in 8-bit integers on MI355X (gfx950), with
 * the norm, activation, bias and residual around them.
 *
 * The reference has no 8-bit path: these stand for its nn.Linear calls (model.py:81-84,107,112-120,
 * 204-207) with the RMSNorm before (model.py:49-55) and the residual add after them (model.py:128-138)
 * in a model whose projections are held in 8 bits.
 *
 * Rows in 8 bits.  A row v of n numbers is held as n int8 and one fp32 scale:
 *   scale = max(max |v|, 2^-100) / 127,   value = round_half_even(v / scale), at most 127 in size
 * (normalised rows: see mi_q8_add_rmsnorm).  A row that holds an infinity or a NaN has scale NaN (and zeros), so that
 * whatever is computed from it is NaN.  The values are laid out for the products: panels of 16 rows,
 *   [ceil(rows / 16)][np / 64][4][16 rows][16 values], np = n rounded up to a multiple of 128,
 * zeros from n on, mi_q8_rows_bytes() bytes, 16-byte aligned; rows past the last keep what they hold.
 *
 * Weights in 8 bits.  int8 [out_features][in_features] and one fp32 scale for each out feature, the
 * values laid out by mi_q8_pack once, as rows are but with zeros past the last.  A gated weight (the gate
 * and up rows of a feed-forward block, gate rows first) is laid out for mi_q8_mlp and used by nothing else.
 *
 * A product is sum_k x[m][k] w[n][k], a whole number in 32 bits (exact, in_features <= 131072), times
 * the two scales in fp32; bias and residual are added in fp32 and the sum is rounded once.
 *
 * Common rules.  dtype: 0 bf16, 1 fp16 (everything that is not int8 or fp32 here).  Row strides are in
 * elements, at least the row's length, any alignment of rows (rows whose addresses are multiples of 16
 * bytes are faster).  Rows of one stride may be columns of one tensor.  Sizes: in_features at most 131072,
 * out_features at most 2^24, rows at most 2^21.
 * All launches are asynchronous on `stream`, allocate nothing and may be captured in a graph.
 * Workspaces: 16-byte aligned, contents arbitrary, not shared by calls that may overlap in time.
 *
 * Status codes as in mi_fa2.h: 0 ok, 1 invalid argument, 2 unsupported, 3 workspace too small,
 * 4 launch failed; mi_q8_last_error() gives the calling thread's last message.
 */
#ifndef MI_Q8_H
#define MI_Q8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MI_Q8_API __attribute__((visibility("default")))

MI_Q8_API const char* mi_q8_last_error(void);

/* Bytes of the values of rows in 8 bits. */
MI_Q8_API size_t mi_q8_rows_bytes(int32_t rows, int32_t n);

/* Rows x [rows, n] in 8 bits. */
MI_Q8_API int mi_q8_quantize(int32_t dtype, const void* x, int64_t x_stride, void* values,
                             float* scale, int32_t rows, int32_t n, void* stream);

/*
 * r = x + y, rounded (y NULL: r is x, and residual_out is not used); values and scale are the rows of
 * r * rsqrt(mean(r^2) + eps) * weight in 8 bits, taken in fp32 without a rounding in between.
 * The largest |r * weight| counts as at least 2^-100.  The mean is fp32's, as mi_fa2_add_rmsnorm's is: of a finite row
 * whose squares pass fp32 (bf16 numbers of 1.8e19 and more) the scale is 0, and the row zeros; where mean and eps are 0 the
 * scale is infinite, and the row zeros times that.
 * residual_out may be x or y, and shares nothing with them otherwise.
 */
typedef struct mi_q8_norm_args {
  const void* x;
  int64_t x_stride;
  const void* y;
  int64_t y_stride;
  const void* weight;
  void* residual_out;
  int64_t residual_stride;
  void* values;
  float* scale;
  int32_t dtype, rows, n;
  float eps;
} mi_q8_norm_args;
MI_Q8_API int mi_q8_add_rmsnorm(const mi_q8_norm_args* args, void* stream);

/* out [rows, n] = values * scale, rounded. */
typedef struct mi_q8_dequantize_args {
  const void* values;
  const float* scale;
  void* out;
  int64_t out_stride;
  int32_t dtype, rows, n;
} mi_q8_dequantize_args;
MI_Q8_API int mi_q8_dequantize(const mi_q8_dequantize_args* args, void* stream);

/*
 * A weight's values (int8, rows of in_features, `stride` bytes apart) in the products' layout:
 * mi_q8_packed_bytes() bytes, 16-byte aligned.  gated: out_features is even, gate rows first.
 */
MI_Q8_API size_t mi_q8_packed_bytes(int32_t out_features, int32_t in_features, int32_t gated);
MI_Q8_API int mi_q8_pack(const void* values, int64_t stride, int32_t out_features,
                         int32_t in_features, int32_t gated, void* packed, void* stream);

/*
 * out = [residual +] x W^T [+ bias]: w packed, w_scale [out_features], bias [out_features] or NULL, residual
 * [rows, out_features] or NULL (may be out, and shares nothing with it otherwise).
 *
 * x_scale NULL: x is 16-bit rows [rows, in_features], which the call brings to 8 bits itself, as
 * mi_q8_add_rmsnorm does without y (norm_weight) or as mi_q8_quantize does (norm_weight NULL); out must not
 * overlap x; workspace: mi_q8_linear_workspace_size() bytes (0 for few rows: none is looked at).
 * Otherwise x and x_scale are rows already in 8 bits as those leave them; x_stride, norm_weight, eps and the
 * workspace are not used.
 */
typedef struct mi_q8_linear_args {
  const void* x;
  int64_t x_stride;
  const float* x_scale;
  const void* norm_weight;
  const void* w;
  const float* w_scale;
  const void* bias;
  const void* residual;
  int64_t residual_stride;
  void* out;
  int64_t out_stride;
  void* workspace;
  size_t workspace_bytes;
  int32_t dtype, rows, out_features, in_features;
  float eps;
} mi_q8_linear_args;
MI_Q8_API size_t mi_q8_linear_workspace_size(int32_t rows, int32_t in_features);
MI_Q8_API int mi_q8_linear(const mi_q8_linear_args* args, void* stream);

/*
 * A gated feed-forward block, out = [residual +] a Wd^T with a = silu(g) * u in fp32, held in 8 bits
 * for the second product, and (g | u) = [rmsnorm] x Wgu^T: x, out, residual [rows, hidden], gate_up
 * packed as gated [2 * inter, hidden], down packed [hidden, inter].  out may be x, and
 * residual (and shares nothing with it otherwise).
 */
typedef struct mi_q8_mlp_args {
  const void* x;
  int64_t x_stride;
  const void* norm_weight;
  const void* gate_up;
  const float* gate_up_scale;
  const void* down;
  const float* down_scale;
  const void* residual;
  int64_t residual_stride;
  void* out;
  int64_t out_stride;
  void* workspace;
  size_t workspace_bytes;
  int32_t dtype, rows, hidden, inter;
  float eps;
} mi_q8_mlp_args;
MI_Q8_API size_t mi_q8_mlp_workspace_size(int32_t rows, int32_t hidden, int32_t inter);
MI_Q8_API int mi_q8_mlp(const mi_q8_mlp_args* args, void* stream);

/*
 * The q/k/v projection of a decode step's few rows with what surrounds it, mi_model_qkv_rope's contract on a
 * weight in 8 bits: (q | k | v) = rmsnorm(x) W^T + bias, rounded, w packed [(heads_q + 2 heads_kv) * 128,
 * hidden]; rotated q to q_out [rows, heads_q * 128], rotated k and v to the cache slot of each token (a slot
 * outside [0, num_slots) writes nothing).  rows <= 16, hidden <= 2048; cos, sin [rows, 128]; k_pool, v_pool
 * [num_slots, heads_kv, 128] with these slot and head strides in elements.  Bitwise mi_q8_linear and
 * mi_fa2_rope_kv_write.
 */
typedef struct mi_q8_qkv_rope_args {
  const void* x;
  int64_t x_stride;
  const void* norm_weight;
  const void* w;
  const float* w_scale;
  const void* bias;
  const void* cos;
  const void* sin;
  int64_t cs_stride;
  const int32_t* slot_mapping;
  void* q_out;
  int64_t q_stride;
  void* k_pool;
  void* v_pool;
  int64_t pool_slot_stride, pool_head_stride;
  int32_t dtype, rows, hidden, heads_q, heads_kv, num_slots;
  float eps;
} mi_q8_qkv_rope_args;
MI_Q8_API int mi_q8_qkv_rope(const mi_q8_qkv_rope_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MI_Q8_H */
