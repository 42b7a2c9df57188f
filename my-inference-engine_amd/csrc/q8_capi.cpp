// C ABI of libmi_q8.so: argument checks and launches of the 8-bit projections.  The contract of every
// entry point is in include/mi_q8.h.
#include "mi_q8.h"

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>

#include "q8.h"

namespace {

using mi_fa2::Q8Params;
using mi_fa2::Q8QuantParams;
using mi_fa2::q8_pad;

enum Status { kOk = 0, kInvalid = 1, kUnsupported = 2, kWorkspace = 3, kLaunch = 4 };

thread_local char g_err[256] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int ok() {
  g_err[0] = '\0';
  return kOk;
}

int launched(hipError_t err) {
  if (err != hipSuccess) return fail(kLaunch, "kernel launch failed: %s", hipGetErrorString(err));
  return ok();
}

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The current device's compute units, read once per device.
int compute_units(int* out) {
  static std::atomic<int> known[64];
  int dev = -1;
  *out = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err == hipSuccess && dev >= 0 && dev < 64) *out = known[dev].load(std::memory_order_relaxed);
  if (err == hipSuccess && *out == 0) {
    err = hipDeviceGetAttribute(out, hipDeviceAttributeMultiprocessorCount, dev);
    if (err == hipSuccess && dev < 64) known[dev].store(*out, std::memory_order_relaxed);
  }
  if (err != hipSuccess || *out <= 0)
    return fail(kLaunch, "reading the device's CU count failed: %s", hipGetErrorString(err));
  return kOk;
}

constexpr int32_t kMaxRows = 1 << 21, kMaxOut = 1 << 24, kMaxK = mi_fa2::kQ8MaxK;

int check_dtype(int32_t dtype) {
  if (dtype != 0 && dtype != 1)
    return fail(kUnsupported, "dtype %d is not bf16 (0) or fp16 (1)", dtype);
  return kOk;
}

int check_count(const char* name, int64_t n, int64_t least, int64_t most) {
  if (n < least || n > most)
    return fail(kInvalid, "%s %lld: %lld to %lld", name, (long long)n, (long long)least,
                (long long)most);
  return kOk;
}

int check_ptr(const char* name, const void* p, int align) {
  if (!p) return fail(kInvalid, "%s is NULL", name);
  if (!aligned(p, align)) return fail(kInvalid, "%s is not %d-byte aligned", name, align);
  return kOk;
}

// Rows of 16-bit elements.
int check_rows(const char* name, const void* p, int64_t stride, int64_t width) {
  if (int rc = check_ptr(name, p, 2)) return rc;
  if (stride < width || stride >= int64_t(1) << 40)
    return fail(kInvalid, "%s row stride %lld: at least %lld", name, (long long)stride,
                (long long)width);
  return kOk;
}

int check_weight(const char* name, const void* w, const float* scale) {
  if (int rc = check_ptr(name, w, 16)) return rc;
  if (!scale || !aligned(scale, 4)) return fail(kInvalid, "%s_scale is %s", name, scale ? "not 4-byte aligned" : "NULL");
  return kOk;
}

// 16-bit rows as a call's arguments describe them.
struct View {
  const void* at;
  int64_t stride;
  int64_t n;
};

// Whether two views of `rows` rows share an element.  Of one stride: exactly (columns of one tensor do not).
// Else by their extents.
bool overlap(int64_t rows, View a, View b) {
  const int64_t d = ((intptr_t)b.at - (intptr_t)a.at) / 2;   // elements from a to b
  if (d >= (rows - 1) * a.stride + a.n || -d >= (rows - 1) * b.stride + b.n) return false;
  const int64_t s = a.stride;
  if (rows == 1 || s != b.stride) return true;
  int64_t q = d / s, e = d % s;   // b's row j begins e elements into a's row q + j
  if (e < 0) --q, e += s;
  return (e < a.n && std::abs(q) < rows) || (e + b.n > s && std::abs(q + 1) < rows);
}

// `out` is `in` itself or shares nothing with it.
int check_in_place(const char* in_name, const char* out_name, int64_t rows, View in, View out) {
  if (in.at == out.at && (rows == 1 || in.stride == out.stride)) return kOk;
  if (!overlap(rows, in, out)) return kOk;
  return fail(kInvalid, "%s overlaps %s, and is not the same rows", out_name, in_name);
}

int check_out(const void* residual, int64_t residual_stride, void* out, int64_t out_stride, int64_t rows,
              int32_t n) {
  if (residual)
    if (int rc = check_rows("residual", residual, residual_stride, n)) return rc;
  if (int rc = check_rows("out", out, out_stride, n)) return rc;
  if (!residual) return kOk;
  return check_in_place("residual", "out", rows, {residual, residual_stride, n}, {out, out_stride, n});
}

// A workspace's parts, each at a multiple of 256 bytes.
struct Space {
  size_t total = 0;
  size_t take(size_t bytes) {
    const size_t at = total;
    total += (bytes + 255) & ~size_t(255);
    return at;
  }
};

// Rows in 8 bits in a workspace.
struct RowsSpace {
  size_t values, scale;
  RowsSpace(Space& s, int32_t rows, int32_t n)
      : values(s.take((size_t)(((int64_t)rows + 15) / 16 * 16) * q8_pad(n))), scale(s.take((size_t)rows * 4)) {}
};

int check_workspace(const void* ws, size_t have, size_t need) {
  if (need == 0) return kOk;
  if (int rc = check_ptr("workspace", ws, 16)) return rc;
  if (have < need) return fail(kWorkspace, "workspace of %zu bytes needed, %zu given", need, have);
  return kOk;
}

int quantize(int dtype, const void* x, int64_t x_stride, const void* y, int64_t y_stride,
             const void* norm_weight, float eps, void* r, int64_t r_stride, void* values,
             float* scale, int32_t rows, int32_t n, void* stream) {
  Q8QuantParams p{};
  p.x = x;
  p.x_st = x_stride;
  p.y = static_cast<const uint16_t*>(y);
  p.y_st = y_stride;
  p.norm_w = static_cast<const uint16_t*>(norm_weight);
  p.eps = eps;
  p.r_out = static_cast<uint16_t*>(r);
  p.r_st = r_stride;
  p.q = static_cast<int8_t*>(values);
  p.scale = scale;
  p.M = rows;
  p.n = n;
  p.np = q8_pad(n);
  return launched(mi_fa2::launch_q8_quant(p, dtype, norm_weight ? mi_fa2::kQ8Norm : mi_fa2::kQ8Plain,
                                          reinterpret_cast<hipStream_t>(stream)));
}

// A product's operands but for its rows.
Q8Params operands(const void* w, const float* w_scale, const void* bias, const void* res,
                  int64_t res_stride, void* out, int64_t out_stride, int32_t rows,
                  int32_t out_features, int32_t in_features, bool gated) {
  Q8Params p{};
  p.w = static_cast<const int8_t*>(w);
  p.w_scale = w_scale;
  p.bias = static_cast<const uint16_t*>(bias);
  p.res = static_cast<const uint16_t*>(res);
  p.res_st = res_stride;
  p.out = out;
  p.out_st = out_stride;
  p.M = rows;
  p.N = out_features;
  p.K = in_features;
  p.Kp = q8_pad(in_features);
  p.panels = mi_fa2::q8_panels(gated ? 2 * out_features : out_features, gated);
  return p;
}

// The product of rows in 8 bits.
int product(Q8Params p, int dtype, bool gated, const void* values, const float* scale, void* stream) {
  p.x = values;
  p.x_scale = scale;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const mi_fa2::Q8Plan plan = mi_fa2::q8_plan(p.M, p.panels, p.Kp);
  switch (plan.kernel) {
    case mi_fa2::kQ8FewRows: {
      int cus = 0;
      if (int rc = compute_units(&cus)) return rc;
      return launched(mi_fa2::launch_q8_rows(p, dtype, gated, mi_fa2::kQ8Rows, cus, st));
    }
    case mi_fa2::kQ8Tile32x32:
    case mi_fa2::kQ8Tile32x64:
    case mi_fa2::kQ8Tile64x64: return launched(mi_fa2::launch_q8_tile(p, plan, dtype, gated, st));
    default: return launched(mi_fa2::launch_q8_gemm(p, plan, dtype, gated, st));
  }
}

// The product of 16-bit rows, brought to 8 bits in the same launch where the few-row kernel does that,
// else before it in the workspace.
bool fused(int32_t rows, int32_t in) {
  return rows <= mi_fa2::kQ8FusedMax && q8_pad(in) <= mi_fa2::kQ8KeepK;
}
int product_of(Q8Params p, int dtype, bool gated, const void* x, int64_t x_stride,
               const void* norm_weight, float eps, const RowsSpace& r, char* ws, void* stream) {
  if (fused(p.M, p.K)) {
    p.x = x;
    p.x_st = x_stride;
    p.norm_w = static_cast<const uint16_t*>(norm_weight);
    p.eps = eps;
    int cus = 0;
    if (int rc = compute_units(&cus)) return rc;
    return launched(mi_fa2::launch_q8_rows(p, dtype, gated, norm_weight ? mi_fa2::kQ8Norm : mi_fa2::kQ8Plain,
                                           cus, reinterpret_cast<hipStream_t>(stream)));
  }
  float* scale = reinterpret_cast<float*>(ws + r.scale);
  if (int rc = quantize(dtype, x, x_stride, nullptr, 0, norm_weight, eps, nullptr, 0, ws + r.values,
                        scale, p.M, p.K, stream))
    return rc;
  return product(p, dtype, gated, ws + r.values, scale, stream);
}

struct LinearSpace {
  Space s;
  RowsSpace x;
  LinearSpace(int32_t rows, int32_t in_features) : x(s, rows, in_features) {}
};

struct MlpSpace {
  Space s;
  RowsSpace x, a;
  size_t act;
  int64_t act_stride;
  MlpSpace(int32_t rows, int32_t hidden, int32_t inter)
      : x(s, rows, hidden), a(s, rows, inter), act(0), act_stride(((int64_t)inter + 7) / 8 * 8) {
    act = s.take((size_t)rows * act_stride * 4);
  }
};

}  // namespace

extern "C" {

const char* mi_q8_last_error(void) { return g_err; }

size_t mi_q8_rows_bytes(int32_t rows, int32_t n) {
  if (rows <= 0 || n <= 0 || rows > kMaxRows || n > kMaxK) return 0;
  return (size_t)((rows + 15) / 16 * 16) * q8_pad(n);
}

int mi_q8_quantize(int32_t dtype, const void* x, int64_t x_stride, void* values, float* scale,
                   int32_t rows, int32_t n, void* stream) {
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_count("rows", rows, 0, kMaxRows)) return rc;
  if (int rc = check_count("n", n, 1, kMaxK)) return rc;
  if (rows == 0) return ok();
  if (int rc = check_rows("x", x, x_stride, n)) return rc;
  if (int rc = check_ptr("values", values, 16)) return rc;
  if (int rc = check_ptr("scale", scale, 4)) return rc;
  return quantize(dtype, x, x_stride, nullptr, 0, nullptr, 0.f, nullptr, 0, values, scale, rows, n,
                  stream);
}

int mi_q8_add_rmsnorm(const mi_q8_norm_args* args, void* stream) {
  if (!args) return fail(kInvalid, "args is NULL");
  const mi_q8_norm_args& a = *args;
  if (int rc = check_dtype(a.dtype)) return rc;
  if (int rc = check_count("rows", a.rows, 0, kMaxRows)) return rc;
  if (int rc = check_count("n", a.n, 1, kMaxK)) return rc;
  if (a.rows == 0) return ok();
  if (int rc = check_rows("x", a.x, a.x_stride, a.n)) return rc;
  if (a.y) {
    if (int rc = check_rows("y", a.y, a.y_stride, a.n)) return rc;
    if (int rc = check_rows("residual_out", a.residual_out, a.residual_stride, a.n)) return rc;
    const View r{a.residual_out, a.residual_stride, a.n};
    if (int rc = check_in_place("x", "residual_out", a.rows, {a.x, a.x_stride, a.n}, r)) return rc;
    if (int rc = check_in_place("y", "residual_out", a.rows, {a.y, a.y_stride, a.n}, r)) return rc;
  }
  if (int rc = check_ptr("weight", a.weight, 2)) return rc;
  if (int rc = check_ptr("values", a.values, 16)) return rc;
  if (int rc = check_ptr("scale", a.scale, 4)) return rc;
  return quantize(a.dtype, a.x, a.x_stride, a.y, a.y_stride, a.weight, a.eps, a.residual_out,
                  a.residual_stride, a.values, a.scale, a.rows, a.n, stream);
}

int mi_q8_dequantize(const mi_q8_dequantize_args* args, void* stream) {
  if (!args) return fail(kInvalid, "args is NULL");
  const mi_q8_dequantize_args& a = *args;
  if (int rc = check_dtype(a.dtype)) return rc;
  if (int rc = check_count("rows", a.rows, 0, kMaxRows)) return rc;
  if (int rc = check_count("n", a.n, 1, kMaxK)) return rc;
  if (a.rows == 0) return ok();
  if (int rc = check_ptr("values", a.values, 16)) return rc;
  if (int rc = check_ptr("scale", a.scale, 4)) return rc;
  if (int rc = check_rows("out", a.out, a.out_stride, a.n)) return rc;
  mi_fa2::Q8DequantParams p{static_cast<const int8_t*>(a.values), a.scale, static_cast<uint16_t*>(a.out),
                            a.out_stride, a.rows, a.n, q8_pad(a.n)};
  return launched(
      mi_fa2::launch_q8_dequant(p, a.dtype, reinterpret_cast<hipStream_t>(stream)));
}

size_t mi_q8_packed_bytes(int32_t out_features, int32_t in_features, int32_t gated) {
  if (out_features <= 0 || in_features <= 0 || out_features > kMaxOut || in_features > kMaxK) return 0;
  return (size_t)mi_fa2::q8_panels(out_features, gated != 0) * 16 * q8_pad(in_features);
}

int mi_q8_pack(const void* values, int64_t stride, int32_t out_features, int32_t in_features,
               int32_t gated, void* packed, void* stream) {
  if (int rc = check_count("out features", out_features, 1, kMaxOut)) return rc;
  if (int rc = check_count("in features", in_features, 1, kMaxK)) return rc;
  if (gated && out_features % 2)
    return fail(kInvalid, "out features %d of a gated weight: gate and up rows", out_features);
  if (int rc = check_ptr("values", values, 1)) return rc;
  if (stride < in_features || stride >= int64_t(1) << 40)
    return fail(kInvalid, "values row stride %lld: at least %d", (long long)stride, in_features);
  if (int rc = check_ptr("packed", packed, 16)) return rc;
  mi_fa2::Q8PackParams p{};
  p.values = static_cast<const int8_t*>(values);
  p.st = stride;
  p.packed = static_cast<int8_t*>(packed);
  p.N = out_features;
  p.K = in_features;
  p.Kp = q8_pad(in_features);
  p.panels = mi_fa2::q8_panels(out_features, gated != 0);
  p.gated = gated != 0;
  p.wide = aligned(values, 16) && stride % 16 == 0;
  return launched(mi_fa2::launch_q8_pack(p, reinterpret_cast<hipStream_t>(stream)));
}

size_t mi_q8_linear_workspace_size(int32_t rows, int32_t in_features) {
  if (rows <= 0 || in_features <= 0 || in_features > kMaxK || fused(rows, in_features)) return 0;
  return LinearSpace(rows, in_features).s.total;
}

int mi_q8_linear(const mi_q8_linear_args* args, void* stream) {
  if (!args) return fail(kInvalid, "args is NULL");
  const mi_q8_linear_args& a = *args;
  if (int rc = check_dtype(a.dtype)) return rc;
  if (int rc = check_count("rows", a.rows, 0, kMaxRows)) return rc;
  if (int rc = check_count("out features", a.out_features, 1, kMaxOut)) return rc;
  if (int rc = check_count("in features", a.in_features, 1, kMaxK)) return rc;
  if (a.rows == 0) return ok();
  if (a.x_scale) {
    if (int rc = check_ptr("x", a.x, 16)) return rc;
    if (int rc = check_ptr("x_scale", a.x_scale, 4)) return rc;
  } else {
    if (int rc = check_rows("x", a.x, a.x_stride, a.in_features)) return rc;
    if (a.norm_weight)
      if (int rc = check_ptr("norm_weight", a.norm_weight, 2)) return rc;
  }
  if (int rc = check_weight("w", a.w, a.w_scale)) return rc;
  if (a.bias)
    if (int rc = check_ptr("bias", a.bias, 2)) return rc;
  if (int rc = check_out(a.residual, a.residual_stride, a.out, a.out_stride, a.rows, a.out_features)) return rc;
  const Q8Params p = operands(a.w, a.w_scale, a.bias, a.residual, a.residual_stride, a.out, a.out_stride,
                              a.rows, a.out_features, a.in_features, false);
  if (a.x_scale) return product(p, a.dtype, false, a.x, a.x_scale, stream);
  if (overlap(a.rows, {a.x, a.x_stride, a.in_features}, {a.out, a.out_stride, a.out_features}))
    return fail(kInvalid, "out overlaps x");
  const LinearSpace sp(a.rows, a.in_features);
  if (int rc = check_workspace(a.workspace, a.workspace_bytes,
                               fused(a.rows, a.in_features) ? 0 : sp.s.total))
    return rc;
  return product_of(p, a.dtype, false, a.x, a.x_stride, a.norm_weight, a.eps, sp.x,
                    static_cast<char*>(a.workspace), stream);
}

size_t mi_q8_mlp_workspace_size(int32_t rows, int32_t hidden, int32_t inter) {
  if (rows <= 0 || hidden <= 0 || inter <= 0 || hidden > kMaxK || inter > kMaxK) return 0;
  return MlpSpace(rows, hidden, inter).s.total;
}

int mi_q8_mlp(const mi_q8_mlp_args* args, void* stream) {
  if (!args) return fail(kInvalid, "args is NULL");
  const mi_q8_mlp_args& a = *args;
  if (int rc = check_dtype(a.dtype)) return rc;
  if (int rc = check_count("rows", a.rows, 0, kMaxRows)) return rc;
  if (int rc = check_count("hidden", a.hidden, 1, kMaxK)) return rc;
  if (int rc = check_count("inter", a.inter, 1, kMaxK)) return rc;
  if (a.rows == 0) return ok();
  if (int rc = check_rows("x", a.x, a.x_stride, a.hidden)) return rc;
  if (a.norm_weight)
    if (int rc = check_ptr("norm_weight", a.norm_weight, 2)) return rc;
  if (int rc = check_weight("gate_up", a.gate_up, a.gate_up_scale)) return rc;
  if (int rc = check_weight("down", a.down, a.down_scale)) return rc;
  if (int rc = check_out(a.residual, a.residual_stride, a.out, a.out_stride, a.rows, a.hidden)) return rc;
  const MlpSpace sp(a.rows, a.hidden, a.inter);
  if (int rc = check_workspace(a.workspace, a.workspace_bytes, sp.s.total)) return rc;
  char* ws = static_cast<char*>(a.workspace);
  if (int rc = product_of(operands(a.gate_up, a.gate_up_scale, nullptr, nullptr, 0, ws + sp.act,
                                   sp.act_stride, a.rows, a.inter, a.hidden, true),
                          a.dtype, true, a.x, a.x_stride, a.norm_weight, a.eps, sp.x, ws, stream))
    return rc;
  Q8Params d = operands(a.down, a.down_scale, nullptr, a.residual, a.residual_stride, a.out,
                        a.out_stride, a.rows, a.hidden, a.inter, false);
  if (a.rows <= mi_fa2::kQ8FloatMax && d.Kp <= mi_fa2::kQ8FloatK) {
    d.x = ws + sp.act;
    d.x_st = sp.act_stride;
    int cus = 0;
    if (int rc = compute_units(&cus)) return rc;
    return launched(mi_fa2::launch_q8_rows(d, a.dtype, false, mi_fa2::kQ8Float, cus,
                                           reinterpret_cast<hipStream_t>(stream)));
  }
  float* a_scale = reinterpret_cast<float*>(ws + sp.a.scale);
  Q8QuantParams q{};
  q.x = ws + sp.act;
  q.x_st = sp.act_stride;
  q.q = reinterpret_cast<int8_t*>(ws + sp.a.values);
  q.scale = a_scale;
  q.M = a.rows;
  q.n = a.inter;
  q.np = q8_pad(a.inter);
  if (int rc = launched(mi_fa2::launch_q8_quant(q, a.dtype, mi_fa2::kQ8Float,
                                                reinterpret_cast<hipStream_t>(stream))))
    return rc;
  return product(d, a.dtype, false, ws + sp.a.values, a_scale, stream);
}

int mi_q8_qkv_rope(const mi_q8_qkv_rope_args* args, void* stream) {
  if (!args) return fail(kInvalid, "args is NULL");
  const mi_q8_qkv_rope_args& a = *args;
  if (int rc = check_dtype(a.dtype)) return rc;
  if (int rc = check_count("rows", a.rows, 0, mi_fa2::kQ8FusedMax)) return rc;
  if (int rc = check_count("hidden", a.hidden, 1, mi_fa2::kQ8KeepK)) return rc;
  if (int rc = check_count("heads_q", a.heads_q, 1, 4096)) return rc;
  if (int rc = check_count("heads_kv", a.heads_kv, 1, 4096)) return rc;
  if (int rc = check_count("num_slots", a.num_slots, 0, INT32_MAX)) return rc;
  if (a.rows == 0) return ok();
  const int d = mi_fa2::kHeadDim;
  if (int rc = check_rows("x", a.x, a.x_stride, a.hidden)) return rc;
  if (int rc = check_ptr("norm_weight", a.norm_weight, 2)) return rc;
  if (int rc = check_weight("w", a.w, a.w_scale)) return rc;
  if (a.bias)
    if (int rc = check_ptr("bias", a.bias, 2)) return rc;
  if (int rc = check_rows("cos", a.cos, a.cs_stride, d)) return rc;
  if (int rc = check_rows("sin", a.sin, a.cs_stride, d)) return rc;
  if (int rc = check_ptr("slot_mapping", a.slot_mapping, 4)) return rc;
  if (int rc = check_rows("q_out", a.q_out, a.q_stride, (int64_t)a.heads_q * d)) return rc;
  if (int rc = check_ptr("k_pool", a.k_pool, 2)) return rc;
  if (int rc = check_ptr("v_pool", a.v_pool, 2)) return rc;
  if (a.pool_slot_stride < d || a.pool_head_stride < d)
    return fail(kInvalid, "pool strides %lld, %lld: at least %d", (long long)a.pool_slot_stride,
                (long long)a.pool_head_stride, d);
  if (overlap(a.rows, {a.x, a.x_stride, a.hidden}, {a.q_out, a.q_stride, a.heads_q * d}))
    return fail(kInvalid, "q_out overlaps x");
  Q8Params p = operands(a.w, a.w_scale, a.bias, nullptr, 0, a.q_out, a.q_stride, a.rows,
                        (a.heads_q + 2 * a.heads_kv) * d, a.hidden, false);
  p.x = a.x;
  p.x_st = a.x_stride;
  p.norm_w = static_cast<const uint16_t*>(a.norm_weight);
  p.eps = a.eps;
  p.cos = static_cast<const uint16_t*>(a.cos);
  p.sin = static_cast<const uint16_t*>(a.sin);
  p.cs_st = a.cs_stride;
  p.slots = a.slot_mapping;
  p.k_pool = static_cast<uint16_t*>(a.k_pool);
  p.v_pool = static_cast<uint16_t*>(a.v_pool);
  p.pool_st = a.pool_slot_stride;
  p.pool_sh = a.pool_head_stride;
  p.num_slots = a.num_slots;
  p.Hq = a.heads_q;
  p.Hkv = a.heads_kv;
  int cus = 0;
  if (int rc = compute_units(&cus)) return rc;
  return launched(mi_fa2::launch_q8_qkv_rope(p, a.dtype, cus, reinterpret_cast<hipStream_t>(stream)));
}

}  // extern "C"
