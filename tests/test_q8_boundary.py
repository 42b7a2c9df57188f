"""CPU checks of libmi_q8.so: it exports exactly what include/mi_q8.h declares and refuses bad arguments
before touching the GPU, and so do the Python wrappers.  No kernel is launched here."""
import re
import subprocess

import pytest
import torch

from conftest import ROOT
from kernels import q8
from oracle import q8 as o8

HEADER = ROOT / "include" / "mi_q8.h"


def declared_symbols():
    return sorted(set(re.findall(r"MI_Q8_API\s+[\w\s\*]+?\b(mi_q8_\w+)\s*\(", HEADER.read_text())))


def test_library_exports_exactly_the_declared_symbols():
    names = declared_symbols()
    out = subprocess.run(["nm", "-D", "--defined-only", str(q8.LIB_PATH)], capture_output=True,
                         text=True, check=True).stdout
    assert sorted(line.split()[-1] for line in out.splitlines() if " T " in line) == names
    assert set(names) == set(q8.SIGNATURES)
    q8.load()


def last():
    return q8.load().mi_q8_last_error().decode()


def _quantize(**over):
    a = dict(dtype=0, x=16, xs=64, values=16, scale=16, rows=3, n=64)
    a.update(over)
    return q8.load().mi_q8_quantize(*a.values(), None)


def _norm(**over):
    a = dict(x=16, xs=64, y=16, ys=64, weight=16, r=16, rs=64, values=16, scale=16, dtype=0, rows=3, n=64,
             eps=1e-6)
    a.update(over)
    return q8.load().mi_q8_add_rmsnorm(q8.NORM_ARGS.pack(*(v or 0 for v in a.values())), None)


def _dequantize(**over):
    a = dict(values=16, scale=16, out=16, os=64, dtype=0, rows=3, n=64)
    a.update(over)
    return q8.load().mi_q8_dequantize(q8.DEQUANTIZE_ARGS.pack(*(v or 0 for v in a.values())), None)


def _pack(**over):
    a = dict(values=16, stride=64, n=48, k=64, gated=0, packed=16)
    a.update(over)
    return q8.load().mi_q8_pack(*a.values(), None)


def _linear(**over):
    a = dict(x=16, xs=64, scale=None, norm=None, w=16, ws=16, bias=None, res=None, rs=0, out=1 << 30, os=48,
             space=16, size=1 << 30, dtype=0, rows=3, n=48, k=64, eps=0.0)
    a.update(over)
    return q8.load().mi_q8_linear(q8.LINEAR_ARGS.pack(*(v or 0 for v in a.values())), None)


def _matmul(**over):
    return _linear(**{"scale": 16, **over})


def _mlp(**over):
    a = dict(x=16, xs=64, norm=None, gu=16, gus=16, down=16, downs=16, res=None, rs=0, out=1 << 30, os=64,
             space=16, size=1 << 30, dtype=0, rows=3, hidden=64, inter=96, eps=0.0)
    a.update(over)
    return q8.load().mi_q8_mlp(q8.MLP_ARGS.pack(*(v or 0 for v in a.values())), None)


def _qkv(**over):
    a = dict(x=16, xs=64, norm=16, w=16, ws=16, bias=None, cos=16, sin=16, cs=128, slots=16, q=1 << 30, qs=256,
             k=16, v=16, ps=128, ph=128, dtype=0, rows=3, hidden=64, heads_q=2, heads_kv=1, num_slots=32,
             eps=0.0)
    a.update(over)
    return q8.load().mi_q8_qkv_rope(q8.QKV_ARGS.pack(*(v or 0 for v in a.values())), None)


@pytest.mark.parametrize("call,over,status,msg", [
    (f, o, s, m) for f in (_quantize, _norm, _dequantize) for o, s, m in [
        (dict(dtype=2), 2, "dtype"), (dict(rows=-1), 1, "rows"), (dict(rows=(1 << 21) + 1), 1, "rows"),
        (dict(n=0), 1, "n 0"), (dict(n=131073), 1, "131072"), (dict(values=None), 1, "values is NULL"),
        (dict(values=24), 1, "16-byte"), (dict(scale=None), 1, "scale is NULL"),
        (dict(scale=18), 1, "4-byte")]] + [
    (_quantize, dict(x=None), 1, "x is NULL"), (_quantize, dict(xs=63), 1, "x row stride"),
    (_quantize, dict(x=17), 1, "2-byte"), (_norm, dict(x=None), 1, "x is NULL"),
    (_norm, dict(ys=10), 1, "y row stride"), (_norm, dict(r=None), 1, "residual_out is NULL"),
    (_norm, dict(rs=1), 1, "residual_out row stride"), (_norm, dict(weight=None), 1, "weight is NULL"),
    (_dequantize, dict(out=None), 1, "out is NULL"), (_dequantize, dict(os=9), 1, "out row stride"),
    (_pack, dict(n=0), 1, "out features"), (_pack, dict(k=0), 1, "in features"),
    (_pack, dict(k=131073, stride=131073), 1, "in features"), (_pack, dict(stride=63), 1, "stride"),
    (_pack, dict(values=None), 1, "values is NULL"), (_pack, dict(packed=8), 1, "16-byte"),
    (_pack, dict(n=(1 << 24) + 1), 1, "out features"), (_pack, dict(n=47, gated=1), 1, "gated")] + [
    (f, o, s, m) for f in (_matmul, _linear) for o, s, m in [
        (dict(dtype=2), 2, "dtype"), (dict(rows=-1), 1, "rows"), (dict(n=0), 1, "out features"),
        (dict(k=131073, xs=131073) if f is _linear else dict(k=131073), 1, "in features"),
        (dict(w=None), 1, "w is NULL"), (dict(w=8), 1, "16-byte"), (dict(ws=None), 1, "w_scale is NULL"),
        (dict(bias=3), 1, "bias"), (dict(res=16, rs=47), 1, "residual row stride"),
        (dict(out=None), 1, "out is NULL"), (dict(os=47), 1, "out row stride")]] + [
    (_matmul, dict(x=None), 1, "x is NULL"), (_matmul, dict(x=24), 1, "16-byte"),
    (_matmul, dict(scale=18), 1, "x_scale is not 4-byte"),
    (_linear, dict(x=None), 1, "x is NULL"), (_linear, dict(norm=3), 1, "norm_weight"),
    (_linear, dict(out=16), 1, "overlaps"), (_linear, dict(out=16 + 2 * (2 * 64 + 63)), 1, "overlaps"),
    (_linear, dict(x=1 << 30, out=(1 << 30) - 2 * (2 * 48 + 47)), 1, "overlaps"),
    # (x: 3 rows of 64 in a stride of 160; out: 48 columns one before its end, or running into its next row)
    (_linear, dict(x=1024, xs=160, out=1024 + 2 * 63, os=160), 1, "overlaps x"),
    (_linear, dict(x=1024, xs=160, out=1024 + 2 * (160 + 113), os=160), 1, "overlaps x"),
    (_linear, dict(x=1024, xs=160, out=1024 - 2 * 47, os=160), 1, "overlaps x"),
    (_linear, dict(x=1024, xs=160, out=1024 + 2 * (320 + 63), os=160), 1, "overlaps x"),
    (_matmul, dict(res=1 << 30, rs=56, os=48), 1, "out overlaps residual"),
    (_matmul, dict(res=(1 << 30) + 2, rs=48), 1, "out overlaps residual"),
    (_mlp, dict(res=(1 << 30) - 2 * (2 * 64 + 63), rs=64), 1, "out overlaps residual"),
    (_norm, dict(r=18), 1, "residual_out overlaps x"), (_norm, dict(x=4096, r=18), 1, "residual_out overlaps y"),
    (_norm, dict(r=16, rs=80), 1, "residual_out overlaps x"),
    # columns of one tensor: past that check, to the workspace's
    *((_linear, dict(rows=300, x=4096, xs=160, out=4096 + 2 * at, os=160, space=None), 1, "workspace is NULL")
      for at in (64, 112, -48, -96, 160 * 299 + 64, -160 * 299 - 48)),
    *((_linear, dict(rows=300, res=(1 << 30) + at, rs=96, os=96, space=None), 1, "workspace is NULL")
      for at in (0, 96, -96)),
    (_linear, dict(rows=300, space=None), 1, "workspace is NULL"),
    (_linear, dict(rows=300, space=8), 1, "16-byte"), (_linear, dict(rows=300, size=255), 3, "needed"),
    (_qkv, dict(dtype=3), 2, "dtype"), (_qkv, dict(rows=17), 1, "rows"), (_qkv, dict(hidden=2049, xs=2049), 1, "hidden"),
    (_qkv, dict(heads_q=0), 1, "heads_q"), (_qkv, dict(heads_kv=5000), 1, "heads_kv"),
    (_qkv, dict(num_slots=-1), 1, "num_slots"), (_qkv, dict(x=None), 1, "x is NULL"),
    (_qkv, dict(norm=None), 1, "norm_weight is NULL"), (_qkv, dict(w=8), 1, "16-byte"),
    (_qkv, dict(ws=None), 1, "w_scale is NULL"), (_qkv, dict(bias=5), 1, "bias"), (_qkv, dict(cs=127), 1, "cos row"),
    (_qkv, dict(sin=None), 1, "sin is NULL"), (_qkv, dict(slots=None), 1, "slot_mapping is NULL"),
    (_qkv, dict(qs=255), 1, "q_out row"), (_qkv, dict(k=None), 1, "k_pool is NULL"),
    (_qkv, dict(ps=100), 1, "pool strides"), (_qkv, dict(q=16), 1, "q_out overlaps"),
    (_mlp, dict(dtype=7), 2, "dtype"), (_mlp, dict(rows=-2), 1, "rows"), (_mlp, dict(hidden=0), 1, "hidden"),
    (_mlp, dict(inter=0), 1, "inter"), (_mlp, dict(inter=131073), 1, "inter"),
    (_mlp, dict(x=None), 1, "x is NULL"), (_mlp, dict(gu=None), 1, "gate_up is NULL"),
    (_mlp, dict(gus=None), 1, "gate_up_scale is NULL"), (_mlp, dict(down=4), 1, "16-byte"),
    (_mlp, dict(res=16, rs=0), 1, "residual row stride"), (_mlp, dict(os=63), 1, "out row stride"),
    (_mlp, dict(space=None), 1, "workspace is NULL"), (_mlp, dict(size=1000), 3, "needed")])
def test_refusals(call, over, status, msg):
    assert call(**over) == status
    assert msg in last()


def test_arguments_that_are_not_there():
    lib = q8.load()
    for fn in (lib.mi_q8_add_rmsnorm, lib.mi_q8_dequantize, lib.mi_q8_linear, lib.mi_q8_mlp, lib.mi_q8_qkv_rope):
        assert fn(None, None) == 1 and "args is NULL" in last()


STRUCTS = """
#include <stdio.h>
#include "mi_q8.h"
int main() {
  printf("%zu %zu %zu %zu %zu\\n", sizeof(mi_q8_dequantize_args), sizeof(mi_q8_norm_args), sizeof(mi_q8_linear_args),
         sizeof(mi_q8_mlp_args), sizeof(mi_q8_qkv_rope_args));
  printf("%zu %zu %zu %zu %zu\\n", offsetof(mi_q8_dequantize_args, n), offsetof(mi_q8_norm_args, eps),
         offsetof(mi_q8_linear_args, eps), offsetof(mi_q8_mlp_args, eps), offsetof(mi_q8_qkv_rope_args, eps));
}
"""


def test_argument_structs_are_the_headers(tmp_path):
    (tmp_path / "s.c").write_text(STRUCTS)
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    sizes, ends = (list(map(int, line.split())) for line in subprocess.run(
        [str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.splitlines())
    for st, size, end in zip((q8.DEQUANTIZE_ARGS, q8.NORM_ARGS, q8.LINEAR_ARGS, q8.MLP_ARGS, q8.QKV_ARGS), sizes, ends):
        assert st.size == end + 4 and st.size <= size < st.size + 8   # (the struct ends aligned)


def test_empty_calls_are_no_ops():
    for call in (_quantize, _norm, _dequantize, _matmul, _linear, _mlp, _qkv):
        assert call(rows=0) == 0 and last() == ""


def test_sizes():
    lib = q8.load()
    for rows, n in ((1, 1), (16, 127), (17, 128), (33, 129), (1 << 21, 131072)):
        assert lib.mi_q8_rows_bytes(rows, n) == q8.rows_bytes(rows, n) == -(-rows // 16) * 16 * (-(-n // 128) * 128)
    assert lib.mi_q8_rows_bytes(0, 5) == lib.mi_q8_rows_bytes(5, 0) == 0
    for n, k, gated in ((1, 1, 0), (2, 1, 1), (16, 64, 0), (17, 129, 0), (34, 129, 1), (2048, 1536, 1)):
        want = o8.packed(torch.zeros(n, k, dtype=torch.int8), gated).numel()
        assert lib.mi_q8_packed_bytes(n, k, gated) == want
    assert lib.mi_q8_packed_bytes(0, 5, 0) == 0 and lib.mi_q8_packed_bytes(5, 131073, 0) == 0
    for rows in (300, 5000):
        # rows in 8 bits and their scales; the feed-forward block's activation in fp32 and 8 bits beside
        assert lib.mi_q8_linear_workspace_size(rows, 1001) >= rows * (1024 + 4)
        assert lib.mi_q8_mlp_workspace_size(rows, 1536, 8960) >= rows * (1536 + 8960 * 5 + 8)
    assert lib.mi_q8_linear_workspace_size(0, 5) == 0 and lib.mi_q8_mlp_workspace_size(1, 0, 5) == 0
    # sizes past 32 bits
    assert lib.mi_q8_mlp_workspace_size(1 << 21, 1536, 8960) > (1 << 21) * 8960 * 5
    assert lib.mi_q8_packed_bytes(1 << 24, 131072, 0) == 1 << 41


def test_wrappers_refuse():
    x, w = torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(16, 64, dtype=torch.int8)
    with pytest.raises(AssertionError):
        q8.Weight(w, torch.ones(16))
    with pytest.raises(AssertionError):
        q8.quantize_weight(x)
    with pytest.raises(AssertionError):
        q8.quantize(x)
    with pytest.raises(AssertionError):
        q8.add_rmsnorm(x, x[0], 1e-6)
    with pytest.raises(AssertionError):
        q8.linear(x, w)
    with pytest.raises(AssertionError):
        q8.mlp(x, w, w)
