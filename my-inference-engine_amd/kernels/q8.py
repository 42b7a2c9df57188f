"""A decoder layer's projections in 8 bits on the HIP kernels (csrc/q8_quant.hip, csrc/q8_rows.hip, through
libmi_q8.so, the C ABI in include/mi_q8.h).

  Weight, quantize_weight   a projection's weight in 8 bits, one scale for each out feature
  quantize, add_rmsnorm     rows of activations in 8 bits, one scale each (Rows)
  linear                    [residual +] ([rmsnorm] x) W^T [+ bias]
  mlp                       [residual +] SwiGLU feed-forward block of [rmsnorm] x
  qkv_rope                  rmsnorm, q/k/v projection, rotary embedding and the paged cache write

They stand beside kernels.few_rows and kernels.model_ops for a model whose projections are held in 8 bits
(Qwen2ForCausalLM.quantize_), and take any number of rows.  The reference has no such path; what surrounds the
products is its model.py:49-55,81-84,107,112-138,204-207.

A row of n numbers v is held as round(v / scale) with scale = max|v| / 127; a row with an infinity or a NaN has
scale NaN, and so is everything computed from it.  A norm's mean is taken in fp32, as kernels.model_ops takes it: of a
finite row whose squares pass that (bf16, 1.8e19 and more) it is infinite and the row comes out as zeros.  Inference
only: no gradient is recorded.  Products are whole numbers, exact in 32 bits; scales, bias and residual are applied in
fp32 and the result is rounded once.  No CPU path and no fallback: a missing library or a call that the kernels do not
take raises.
"""
import ctypes
import os
import struct
from pathlib import Path

import torch

from . import _lib
from .fa2 import _MEMO_MAX
from .rope import HEAD_DIM, rope_kv_write

LIB_PATH = Path(os.environ.get("MI_Q8_LIB", Path(__file__).resolve().parent / "libmi_q8.so"))

MAX_ROWS = 1 << 21
MAX_IN = 131072      # 128 * 127 * in stays below 2^31
MAX_OUT = 1 << 24
FUSED_ROWS, FUSED_IN = 16, 2048   # of qkv_rope in one launch

_p, _i32, _i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
_sz, _args = ctypes.c_size_t, ctypes.c_char_p
# name -> (restype, argtypes); mirrors include/mi_q8.h
SIGNATURES = {
    "mi_q8_last_error": (ctypes.c_char_p, []),
    "mi_q8_rows_bytes": (_sz, [_i32, _i32]),
    "mi_q8_quantize": (_i32, [_i32, _p, _i64, _p, _p, _i32, _i32, _p]),
    "mi_q8_add_rmsnorm": (_i32, [_args, _p]),
    "mi_q8_dequantize": (_i32, [_args, _p]),
    "mi_q8_packed_bytes": (_sz, [_i32, _i32, _i32]),
    "mi_q8_pack": (_i32, [_p, _i64, _i32, _i32, _i32, _p, _p]),
    "mi_q8_linear_workspace_size": (_sz, [_i32, _i32]),
    "mi_q8_linear": (_i32, [_args, _p]),
    "mi_q8_mlp_workspace_size": (_sz, [_i32, _i32, _i32]),
    "mi_q8_mlp": (_i32, [_args, _p]),
    "mi_q8_qkv_rope": (_i32, [_args, _p]),
}
# the argument structs, packed in one go: a call of 18 arguments costs ctypes 1.9 us, this 0.6
NORM_ARGS = struct.Struct("@PqPqPPqPPiiif")
DEQUANTIZE_ARGS = struct.Struct("@PPPqiii")
LINEAR_ARGS = struct.Struct("@PqPPPPPPqPqPNiiiif")
QKV_ARGS = struct.Struct("@PqPPPPPPqPPqPPqqiiiiiif")
MLP_ARGS = struct.Struct("@PqPPPPPPqPqPNiiiif")

_library = None


def load():
    """Load libmi_q8.so once; raise if it is missing."""
    global _library
    if _library is None:
        if not LIB_PATH.exists():
            raise ImportError(
                f"{LIB_PATH} not found: build it with `python my-inference-engine_amd/build_lib.py`")
        lib = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _library = lib
    return _library


def check(status):
    if status != _lib.OK:
        raise _lib.MiFa2Error(f"libmi_q8 status {status}: {load().mi_q8_last_error().decode()}")


def call(device, fn, *args):
    """fn(*args, stream) on the device's current stream; raises what it reports."""
    if device == torch._C._cuda_getDevice():
        check(fn(*args, torch._C._cuda_getCurrentRawStream(device)))
        return
    with _lib.on_device(torch.device("cuda", device)) as stream:
        check(fn(*args, stream))


def rows_bytes(rows, n):
    """Bytes of the values of rows in 8 bits: panels of 16 rows, n rounded up to 128."""
    return -(-rows // 16) * 16 * (-(-n // 128) * 128)


class Weight:
    """A projection's weight in 8 bits: values [out, in] int8 and scale [out] fp32 (weight = values *
    scale[:, None]), laid out for the kernels once.  gated: the gate and up rows of a feed-forward block,
    gate rows first, which only `mlp` takes.  The values are copied, the scale is kept as it is."""
    __slots__ = ("data", "scale", "out_features", "in_features", "gated", "sig")

    def __init__(self, values, scale, gated=False):
        assert values.is_cuda and values.dtype == torch.int8 and values.dim() == 2, \
            "values: an int8 GPU tensor [out, in]"
        n, k = values.shape
        assert 1 <= n <= MAX_OUT and 1 <= k <= MAX_IN, \
            f"a weight of 1 to {MAX_OUT} out features and 1 to {MAX_IN} in features"
        assert values.stride(1) == 1 or k == 1, "values: unit column stride"
        assert scale.device == values.device and scale.dtype == torch.float32, \
            f"scale: fp32 on {values.device}"
        assert scale.shape == (n,) and scale.is_contiguous(), f"scale: contiguous, of {n}"
        gated = bool(gated)
        assert not (gated and n % 2), "a gated weight has as many gate as up rows"
        lib = load()
        data = torch.empty(lib.mi_q8_packed_bytes(n, k, gated), dtype=torch.int8, device=values.device)
        call(values.device.index, lib.mi_q8_pack, values.data_ptr(),
             values.stride(0) if n > 1 else k, n, k, gated, data.data_ptr())
        self._hold(data, scale, n, k, gated)

    def _hold(self, data, scale, n, k, gated):
        self.data, self.scale, self.out_features, self.in_features, self.gated = data, scale, n, k, gated
        self.sig = (n, k, gated, scale.device)   # what a call's plan depends on

    def __reduce__(self):   # copied and saved as its two tensors, wherever those come back
        return _held, (self.data, self.scale, self.out_features, self.in_features, self.gated)

    @property
    def device(self):
        return self.scale.device


def _held(*parts):
    w = object.__new__(Weight)
    w._hold(*parts)
    return w


def quantize_weight(weight, gated=False):
    """weight [out, in] (bf16 or fp16) in 8 bits, every row by its largest magnitude."""
    rows = quantize(weight)
    return Weight(rows.values, rows.scale, gated)


class Rows:
    """Rows in 8 bits as the kernels read them: data (their values, in panels of 16 rows: `values` has them as
    [rows, n]), scale [rows] fp32, n the row's length and dtype the type of the rows that they stand for."""
    __slots__ = ("data", "scale", "n", "dtype")

    def __init__(self, data, scale, n, dtype):
        assert 1 <= n <= MAX_IN and scale.dim() == 1 and scale.shape[0] <= MAX_ROWS, \
            f"at most {MAX_ROWS} rows of 1 to {MAX_IN}"
        assert data.dtype == torch.int8 and data.is_contiguous() and data.numel() == rows_bytes(scale.shape[0], n), \
            f"data: contiguous int8 of {rows_bytes(scale.shape[0], n)}"
        assert scale.dtype == torch.float32 and scale.is_contiguous(), "scale: contiguous fp32"
        assert dtype in _lib.DTYPES, "dtype: bf16 or fp16"
        assert data.is_cuda and data.device == scale.device, "data and scale on one GPU"
        self._hold(data, scale, n, dtype)

    def _hold(self, data, scale, n, dtype):
        self.data, self.scale, self.n, self.dtype = data, scale, n, dtype

    @property
    def values(self):
        """[rows, n] int8."""
        R = self.scale.shape[0]
        np = -(-self.n // 128) * 128
        whole = self.data.view(-1, np // 64, 4, 16, 16).permute(0, 3, 1, 2, 4)
        return whole.reshape(-1, np)[:R, :self.n].contiguous()

    def dequantize(self, out=None):
        """values * scale [rows, n] in dtype."""
        scale, dt = self.scale, self.dtype
        R, dev = scale.shape[0], scale.device
        if out is None:
            out, os_ = torch.empty((R, self.n), device=dev, dtype=dt), self.n
        else:
            _, os_ = _rows(out, "out", dt, dev)
            assert out.shape == (R, self.n), f"out: [{R}, {self.n}]"
        call(dev.index, load().mi_q8_dequantize, DEQUANTIZE_ARGS.pack(
            self.data.data_ptr(), scale.data_ptr(), out.data_ptr(), os_, _lib.DTYPES[dt], R, self.n))
        return out


def _rows(t, name, dtype, device):
    """(address, row stride) of [rows, n] with unit column stride."""
    assert t.device == device and t.dtype == dtype, f"{name}: a {dtype} tensor on {device}"
    assert t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] == 1), \
        f"{name}: [rows, n] with unit column stride"
    # one row: its stride is never used, and torch may report any value there
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _vector(t, name, n, dtype, device):
    assert t.device == device and t.dtype == dtype and t.shape == (n,) and t.is_contiguous(), \
        f"{name}: contiguous {dtype} of {n} on {device}"
    return t.data_ptr()


def _input(x):
    assert x.is_cuda and x.dtype in _lib.DTYPES, "x: a bf16 / fp16 GPU tensor"
    assert x.dim() == 2 and 1 <= x.shape[1] <= MAX_IN and x.shape[0] <= MAX_ROWS, \
        f"x: [rows, n], at most {MAX_ROWS} rows of 1 to {MAX_IN}"
    return x.dtype, x.device


def _empty_rows(R, n, dtype, dev):
    rows = object.__new__(Rows)
    rows._hold(torch.empty(rows_bytes(R, n), dtype=torch.int8, device=dev),
               torch.empty(R, dtype=torch.float32, device=dev), n, dtype)
    return rows


_ROWS_GO = "x: 16-bit rows (rows in 8 bits go to linear)"


def quantize(x):
    """Rows x [rows, n] in 8 bits."""
    assert type(x) is not Rows, _ROWS_GO
    dt, dev = _input(x)
    R, n = x.shape
    xp, xs = _rows(x, "x", dt, dev)
    out = _empty_rows(R, n, dt, dev)
    call(dev.index, load().mi_q8_quantize, _lib.DTYPES[dt], xp, xs, out.data.data_ptr(),
         out.scale.data_ptr(), R, n)
    return out


# What a call's shapes, strides, types and devices decide, checked once per combination.
_PLANS = {}


def _plan(key, make, *args):
    if len(_PLANS) >= _MEMO_MAX:
        _PLANS.clear()
    got = _PLANS[key] = make(*args)
    return got


def _sig(t):
    return (t.shape, t.stride(), t.dtype, t.device) if t is not None else None


def add_rmsnorm(x, weight, eps, y=None, residual_out=None):
    """x [rows, n] (+ y) -> (r, Rows): r = x + y rounded (x itself when y is None), and weight * rmsnorm(r)
    in 8 bits, with no rounding to 16 bits in between.  residual_out may be x or y (in place)."""
    assert type(x) is not Rows, _ROWS_GO
    key = ("norm", x.shape, x.stride(), x.dtype, x.device, _sig(weight), _sig(y), _sig(residual_out))
    plan = _PLANS.get(key)
    if plan is None:
        plan = _plan(key, _norm_plan, x, weight, y, residual_out)
    index, fn, code, R, n, nbytes, xs, ys, rs = plan
    if y is None:
        r, yp, rp = x, 0, 0
    else:
        r = x.new_empty((R, n)) if residual_out is None else residual_out
        yp, rp = y.data_ptr(), r.data_ptr()
    dev = x.device
    rows = object.__new__(Rows)
    # (one allocation of both and views into it are slower: 14.4 -> 16.2 us with `dequantize`)
    rows.data = data = torch.empty(nbytes, dtype=torch.int8, device=dev)
    rows.scale = scale = torch.empty(R, dtype=torch.float32, device=dev)
    rows.n, rows.dtype = n, x.dtype
    call(index, fn, NORM_ARGS.pack(x.data_ptr(), xs, yp, ys, weight.data_ptr(), rp, rs,
                                   data.data_ptr(), scale.data_ptr(), code, R, n, eps))
    return r, rows


def _norm_plan(x, weight, y, residual_out):
    dt, dev = _input(x)
    R, n = x.shape
    _, xs = _rows(x, "x", dt, dev)
    _vector(weight, "weight", n, dt, dev)
    ys, rs = 0, n
    if y is not None:
        _, ys = _rows(y, "y", dt, dev)
        assert y.shape == x.shape, "y: x's shape"
        if residual_out is not None:
            _, rs = _rows(residual_out, "residual_out", dt, dev)
            assert residual_out.shape == x.shape, "residual_out: x's shape"
    else:
        assert residual_out is None, "residual_out goes with y"
    return (dev.index, load().mi_q8_add_rmsnorm, _lib.DTYPES[dt], R, n, rows_bytes(R, n), xs, ys, rs)


def _ends(out, residual, R, N, dt, dev):
    """Row strides of out (None: a new one) and residual (or None) [R, N]."""
    os_, rs = N, 0
    if out is not None:
        _, os_ = _rows(out, "out", dt, dev)
        assert out.shape == (R, N), f"out: [{R}, {N}]"
    if residual is not None:
        _, rs = _rows(residual, "residual", dt, dev)
        assert residual.shape == (R, N), f"residual: [{R}, {N}]"
    return os_, rs


def linear(x, w, bias=None, residual=None, norm_weight=None, eps=0.0, out=None):
    """[residual +] x W^T [+ bias] -> [rows, out]: x [rows, in] (bf16 or fp16; with norm_weight RMS-normalised
    first) or Rows, w a Weight.  residual may be `out` (in place); out shares nothing with x."""
    assert type(w) is Weight, "w: a Weight"
    if type(x) is Rows:
        assert norm_weight is None, "rows in 8 bits are normalised already"
        data, scale = x.data, x.scale
        key = ("rows", x.n, x.dtype, scale.shape, scale.device, w.sig, _sig(bias), _sig(residual), _sig(out))
    else:
        data, scale = x, None
        key = ("linear", x.shape, x.stride(), x.dtype, x.device, w.sig, _sig(bias), _sig(residual), _sig(out),
               _sig(norm_weight))
    plan = _PLANS.get(key)
    if plan is None:
        plan = _plan(key, _linear_plan, x, w, bias, residual, norm_weight, out)
    index, fn, code, dt, shape, K, nbytes, xs, rs, os_ = plan
    if out is None:
        out = torch.empty(shape, dtype=dt, device=data.device)
    # every call has its own (from torch's caching allocator, in stream order): nothing is shared
    ws = torch.empty(nbytes, dtype=torch.uint8, device=data.device) if nbytes else None
    call(index, fn, LINEAR_ARGS.pack(
        data.data_ptr(), xs, scale.data_ptr() if scale is not None else 0,
        norm_weight.data_ptr() if norm_weight is not None else 0, w.data.data_ptr(), w.scale.data_ptr(),
        bias.data_ptr() if bias is not None else 0, residual.data_ptr() if residual is not None else 0,
        rs, out.data_ptr(), os_, ws.data_ptr() if nbytes else 0, nbytes, code, *shape, K, eps))
    return out


def _linear_plan(x, w, bias, residual, norm_weight, out):
    assert not w.gated, "w: a Weight that is not gated"
    N, K = w.out_features, w.in_features
    lib = load()
    if type(x) is Rows:
        dt, dev, R = x.dtype, x.scale.device, x.scale.shape[0]
        assert x.n == K and w.device == dev, f"x: rows of {K} on {w.device}"
        xs = nbytes = 0
    else:
        dt, dev = _input(x)
        R = x.shape[0]
        assert x.shape[1] == K and w.device == dev, f"x: rows of {K} on {w.device}"
        _, xs = _rows(x, "x", dt, dev)
        nbytes = lib.mi_q8_linear_workspace_size(R, K)
        if norm_weight is not None:
            _vector(norm_weight, "norm_weight", K, dt, dev)
    if bias is not None:
        _vector(bias, "bias", N, dt, dev)
    os_, rs = _ends(out, residual, R, N, dt, dev)
    return (dev.index, lib.mi_q8_linear, _lib.DTYPES[dt], dt, (R, N), K, nbytes, xs, rs, os_)


def mlp(x, gate_up, down, residual=None, norm_weight=None, eps=0.0, out=None):
    """[residual +] (silu(g) * u) Wd^T with (g | u) = [rmsnorm] x Wgu^T -> [rows, hidden]: x [rows, hidden],
    gate_up a gated Weight [2 * inter, hidden], down a Weight [hidden, inter].  The activation is held in 8 bits
    too, every row by its largest magnitude.  out may be residual and x."""
    assert type(gate_up) is Weight and type(down) is Weight, "gate_up, down: Weights"
    assert type(x) is not Rows, _ROWS_GO
    key = ("mlp", x.shape, x.stride(), x.dtype, x.device, gate_up.sig, down.sig, _sig(residual),
           _sig(norm_weight), _sig(out))
    plan = _PLANS.get(key)
    if plan is None:
        plan = _plan(key, _mlp_plan, x, gate_up, down, residual, norm_weight, out)
    index, fn, code, R, H, inter, nbytes, xs, rs, os_ = plan
    if out is None:
        out = x.new_empty((R, H))
    # every call has its own (from torch's caching allocator, in stream order): nothing is shared
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    call(index, fn, MLP_ARGS.pack(
        x.data_ptr(), xs, norm_weight.data_ptr() if norm_weight is not None else 0, gate_up.data.data_ptr(),
        gate_up.scale.data_ptr(), down.data.data_ptr(), down.scale.data_ptr(),
        residual.data_ptr() if residual is not None else 0, rs, out.data_ptr(), os_, ws.data_ptr(),
        nbytes, code, R, H, inter, eps))
    return out


def _mlp_plan(x, gate_up, down, residual, norm_weight, out):
    assert gate_up.gated, "gate_up: a gated Weight"
    assert not down.gated, "down: a Weight that is not gated"
    dt, dev = _input(x)
    R, H = x.shape
    inter = down.in_features
    assert gate_up.in_features == H and down.out_features == H, f"weights of hidden size {H}"
    assert gate_up.out_features == 2 * inter, f"gate_up of {2 * inter} rows"
    assert gate_up.device == dev and down.device == dev, f"weights on {dev}"
    _, xs = _rows(x, "x", dt, dev)
    if norm_weight is not None:
        _vector(norm_weight, "norm_weight", H, dt, dev)
    os_, rs = _ends(out, residual, R, H, dt, dev)
    lib = load()
    return (dev.index, lib.mi_q8_mlp, _lib.DTYPES[dt], R, H, inter,
            lib.mi_q8_mlp_workspace_size(R, H, inter), xs, rs, os_)


def qkv_rope(x, norm_weight, eps, w, bias, cos, sin, slot_mapping, k_pool, v_pool, heads_q, heads_kv):
    """x [rows, hidden], w a Weight [(heads_q + 2 heads_kv) * 128, hidden], cos/sin [rows, 128], slot_mapping
    [rows] int32, k_pool/v_pool [slots, heads_kv, 128] (one layer of KVCache.buf).  Returns the rotated queries
    [rows, heads_q * 128]; k and v go to the rows' cache slots (a slot outside the pool: nowhere).  Up to 16 rows
    of a hidden size up to 2048 in one launch, more through `linear` and rope_kv_write (whose rows of cos and sin
    lie at multiples of 16 bytes), bitwise the same."""
    assert type(w) is Weight, "w: a Weight"
    assert type(x) is not Rows, _ROWS_GO
    rows, hidden = x.shape
    if rows > FUSED_ROWS or hidden > FUSED_IN:
        qkv = linear(x, w, bias=bias, norm_weight=norm_weight, eps=eps)
        return rope_kv_write(qkv, cos, sin, slot_mapping, k_pool, v_pool, heads_q, heads_kv)
    key = ("qkv", x.shape, x.stride(), x.dtype, x.device, w.sig, _sig(norm_weight), _sig(bias), _sig(cos),
           _sig(sin), _sig(slot_mapping), _sig(k_pool), _sig(v_pool), heads_q, heads_kv)
    plan = _PLANS.get(key)
    if plan is None:
        plan = _plan(key, _qkv_plan, x, w, norm_weight, bias, cos, sin, slot_mapping, k_pool, v_pool, heads_q,
                     heads_kv)
    index, fn, code, xs, cs, pool_strides, slots, width = plan
    q = x.new_empty((rows, width))
    call(index, fn, QKV_ARGS.pack(
        x.data_ptr(), xs, norm_weight.data_ptr(), w.data.data_ptr(), w.scale.data_ptr(),
        bias.data_ptr() if bias is not None else 0, cos.data_ptr(), sin.data_ptr(), cs,
        slot_mapping.data_ptr(), q.data_ptr(), width, k_pool.data_ptr(), v_pool.data_ptr(), *pool_strides,
        code, rows, hidden, heads_q, heads_kv, slots, eps))
    return q


def _qkv_plan(x, w, norm_weight, bias, cos, sin, slot_mapping, k_pool, v_pool, heads_q, heads_kv):
    dt, dev = _input(x)
    R, H = x.shape
    assert not w.gated and w.device == dev, f"w: a Weight on {dev} that is not gated"
    n_out = (heads_q + 2 * heads_kv) * HEAD_DIM
    assert w.in_features == H and w.out_features == n_out, f"w: [{n_out}, {H}]"
    _, xs = _rows(x, "x", dt, dev)
    _vector(norm_weight, "norm_weight", H, dt, dev)
    if bias is not None:
        _vector(bias, "bias", n_out, dt, dev)
    _, cs = _rows(cos, "cos", dt, dev)
    assert cos.shape == (R, HEAD_DIM) and sin.shape == (R, HEAD_DIM) and _rows(sin, "sin", dt, dev)[1] == cs, \
        f"cos, sin: [{R}, {HEAD_DIM}], alike"
    assert slot_mapping.device == dev and slot_mapping.dtype == torch.int32 and slot_mapping.shape == (R,) \
        and slot_mapping.is_contiguous(), f"slot_mapping: contiguous int32 of {R} on {dev}"
    for pool, name in ((k_pool, "k_pool"), (v_pool, "v_pool")):
        assert pool.device == dev and pool.dtype == dt and pool.dim() == 3 and pool.stride(2) == 1, \
            f"{name}: a {dt} [slots, heads_kv, {HEAD_DIM}] on {dev}"
        assert pool.shape[1:] == (heads_kv, HEAD_DIM), f"{name}: [slots, {heads_kv}, {HEAD_DIM}]"
    assert k_pool.shape == v_pool.shape and k_pool.stride() == v_pool.stride(), "pools of one shape and strides"
    return (dev.index, load().mi_q8_qkv_rope, _lib.DTYPES[dt], xs, cs, k_pool.stride()[:2], k_pool.shape[0],
            heads_q * HEAD_DIM)
