"""CPU checks of libmi_cache.so: it exports exactly what include/mi_cache.h declares and refuses bad
arguments before touching the GPU, and so do the Python wrappers.  No kernel is launched here."""
import ctypes
import re
import subprocess

import pytest
import torch

from conftest import ROOT
from kernels import blocks, shared

HEADER = ROOT / "include" / "mi_cache.h"


def declared_symbols():
    return sorted(set(re.findall(r"MI_CACHE_API\s+[\w\s\*]+?\b(mi_cache_\w+)\s*\(",
                                 HEADER.read_text())))


def test_library_exports_exactly_the_declared_symbols():
    names = declared_symbols()
    out = subprocess.run(["nm", "-D", "--defined-only", str(blocks.LIB_PATH)], capture_output=True,
                         text=True, check=True).stdout
    assert sorted(line.split()[-1] for line in out.splitlines() if " T " in line) == names
    assert set(names) == set(blocks.SIGNATURES)
    blocks.load()


def last():
    return blocks.load().mi_cache_last_error().decode()


def _copy(**over):
    a = dict(src=16, src_plane=1 << 20, src_blocks=64, dst=16, dst_plane=1 << 20, dst_blocks=64,
             planes=2, size=8192, pairs=16, n=3)
    a.update(over)
    return blocks.load().mi_cache_copy_blocks(*a.values(), None)


@pytest.mark.parametrize("over,status,msg", [
    (dict(src=None), 1, "src is NULL"), (dict(dst=None), 1, "dst is NULL"),
    (dict(pairs=None), 1, "pairs is NULL"), (dict(n=-1), 1, "bad counts"),
    (dict(src_blocks=-1), 1, "bad sizes"), (dict(planes=-2), 1, "bad sizes"),
    (dict(size=0), 1, "bad sizes"), (dict(planes=70000), 2, "planes"),
    (dict(src_blocks=129), 1, "do not hold"), (dict(dst_plane=8191, dst_blocks=1), 1, "do not hold"),
    (dict(n=1 << 23), 2, "in one call"),
    (dict(size=(1 << 40) + 1, src_blocks=0, dst_blocks=0), 1, "do not hold"),
])
def test_copy_refuses(over, status, msg):
    assert _copy(**over) == status
    assert msg in last()


def test_empty_calls_are_no_ops():
    assert _copy(n=0, pairs=None) == 0
    assert _copy(planes=0) == 0
    assert _fork(n=0, children=None) == 0
    assert _move(n=0, pairs=None, n_rows=0, rows=None, tables=None, new_ids=None) == 0
    assert _attend(batch=0, n_groups=0) == 0
    assert _attend(total_q=0) == 0


def _fork(**over):
    a = dict(pool=16, plane=1 << 20, blocks=64, planes=2, bs=16, token=512, tables=16, stride=40,
             width=40, lens=16, max_seqs=8, children=16, n=3)
    a.update(over)
    return blocks.load().mi_cache_fork_rows(*a.values(), None)


@pytest.mark.parametrize("over,status,msg", [
    (dict(pool=None), 1, "pool is NULL"), (dict(tables=None), 1, "tables is NULL"),
    (dict(lens=None), 1, "seq_lens is NULL"), (dict(children=None), 1, "children is NULL"),
    (dict(bs=0), 1, "bad block"), (dict(token=0), 1, "bad block"), (dict(stride=39), 1, "bad tables"),
    (dict(width=-1), 1, "bad tables"), (dict(blocks=200), 1, "do not hold"),
    (dict(planes=0), 1, "no planes"), (dict(n=-3), 1, "bad counts"),
])
def test_fork_refuses(over, status, msg):
    assert _fork(**over) == status
    assert msg in last()


def _move(**over):
    a = dict(pool=16, plane=1 << 20, blocks=64, planes=2, size=8192, pairs=16, n=3, tables=16,
             stride=40, width=40, max_seqs=8, rows=16, n_rows=2, new_ids=16)
    a.update(over)
    return blocks.load().mi_cache_move_blocks(*a.values(), None)


@pytest.mark.parametrize("over,status,msg", [
    (dict(pool=None), 1, "pool is NULL"), (dict(tables=None), 1, "tables is NULL"),
    (dict(pairs=None), 1, "pairs is NULL"), (dict(rows=None), 1, "rows is NULL"),
    (dict(new_ids=None), 1, "new_ids is NULL"), (dict(n_rows=-1), 1, "bad counts"),
    (dict(size=-8), 1, "bad sizes"),
])
def test_move_refuses(over, status, msg):
    assert _move(**over) == status
    assert msg in last()


def _attend(**over):
    i64 = lambda *v: (ctypes.c_int64 * len(v))(*v)  # noqa: E731
    a = dict(dtype=0, q=16, k=16, v=16, o=16, lse=None, cu_q=16, table=16, bt_stride=8, kv_lens=16,
             cu_rows=16, prefix=16, n_groups=1, batch=2, total_q=2, heads_q=12, heads_kv=2,
             max_kv=64, d=128, bs=16, num_blocks=10, qs=i64(1536, 128), ps=i64(256, 128),
             os=i64(1536, 128), ls=None, causal=1, scale=0.1, ws=None, ws_bytes=0)
    a.update(over)
    return blocks.load().mi_cache_attend(*a.values(), None)


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


@pytest.mark.parametrize("over,status,msg", [
    (dict(dtype=2), 2, "dtype"), (dict(d=64), 2, "head_dim 64"), (dict(heads_kv=5), 1, "bad sizes"),
    (dict(batch=-1), 1, "bad sizes"), (dict(batch=513), 2, "512"), (dict(total_q=1 << 22), 2, "2^25"),
    (dict(total_q=1 << 21, max_kv=1 << 23), 2, "in one call"), (dict(n_groups=3), 1, "n_groups"),
    (dict(max_kv=-1), 1, "max_kv_len"), (dict(bs=24), 2, "block_size"), (dict(bs=8), 2, "block_size"),
    (dict(num_blocks=-1), 1, "num_blocks"), (dict(scale=0.0), 1, "sm_scale"),
    (dict(scale=float("nan")), 1, "sm_scale"), (dict(cu_q=None), 1, "cu_seqlens_q"),
    (dict(kv_lens=None), 1, "kv_lens"), (dict(cu_rows=None), 1, "cu_rows"),
    (dict(table=None), 1, "block_table"), (dict(q=None), 1, "q is NULL"), (dict(o=24), 1, "aligned"),
    (dict(k=8), 1, "aligned"), (dict(qs=i64(1500, 128)), 1, "multiple of 8"),
    (dict(ps=i64(64, 128)), 1, "slot stride"), (dict(ps=i64(1 << 24, 128)), 2, "slot stride"),
    (dict(lse=16), 1, "lse strides"), (dict(bt_stride=-1), 1, "stride -1"),
])
def test_attend_refuses(over, status, msg):
    assert _attend(**over) == status
    assert msg in last()


def test_wrappers_refuse_cpu_tensors():
    pool = torch.zeros(2, 32, 2, 128, dtype=torch.bfloat16)
    ids = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="GPU"):
        blocks.copy_blocks(pool, pool, ids, 16)
    with pytest.raises(AssertionError, match="GPU"):
        blocks.fork_rows(pool, ids, ids[0], torch.zeros(1, 4, dtype=torch.int32), 16)
    with pytest.raises(AssertionError, match="GPU"):
        blocks.move_blocks(pool, ids, ids, ids, ids[0], 16)
    with pytest.raises(AssertionError, match="GPU"):
        shared.fa2_paged_shared(pool[0], pool[0], pool[0], ids[0], ids, ids[0], 1, ids[0], ids[0])


def _gpu_like(*shape, dtype=torch.bfloat16):
    from test_split_workspace import on_gpu
    return on_gpu(*shape, dtype=dtype)


@pytest.mark.parametrize("make,match", [
    (lambda p: (p, p.float(), 16), "one dtype"),
    (lambda p: (p, _gpu_like(2, 32, 4, 128), 16), "same planes"),
    (lambda p: (p, _gpu_like(3, 32, 2, 128), 16), "same planes"),
    (lambda p: (p[:, :, :1], p[:, :, 1:], 16), "contiguous"),
    (lambda p: (p[..., :64], p[..., 64:], 16), "contiguous"),
    (lambda p: (p, p, 24), "whole blocks"),
    (lambda p: (p, p, 0), "positive int"),
    (lambda p: (p, p, 16.0), "positive int"),
    (lambda p: (p[:1].expand(2, -1, -1, -1), p, 16), "overlap"),
])
def test_copy_blocks_refuses(make, match):
    src, dst, size = make(_gpu_like(2, 32, 2, 128))
    with pytest.raises(AssertionError, match=match):
        blocks.copy_blocks(src, dst, torch.zeros(1, 2, dtype=torch.int32), size)


@pytest.mark.parametrize("pairs", [torch.zeros(1, 2), torch.zeros(2, dtype=torch.int32),
                                   torch.zeros(1, 3, dtype=torch.int32),
                                   torch.zeros(2, 4, dtype=torch.int32)[:, ::2]])
def test_copy_blocks_refuses_pairs(pairs):
    pool = _gpu_like(2, 32, 2, 128)
    with pytest.raises(AssertionError, match="pairs"):
        blocks.copy_blocks(pool, pool, pairs, 16)


def test_workspace():
    size = blocks.load().mi_cache_attend_workspace_size
    # parts of 128 + 2 floats: two columns per (token, head) in either area, 128 for each of 256
    # work-groups and 32 for each of their 2,048 waves; a record of two words for each column of an area
    assert size(64, 12) == (4 * 64 * 12 + 98304) * 520 + 2 * 64 * 12 * 8
    assert size(0, 12) == 0 and size(1 << 22, 12) == 0
    assert _attend() == 3 and "workspace" in last()
    assert _attend(ws=24, ws_bytes=1 << 30) == 3
    assert _attend(ws=16, ws_bytes=size(2, 12) - 1) == 3


def test_attention_refuses_bad_arguments():
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32)  # noqa: E731
    good = dict(q=_gpu_like(3, 12, 128), k_pool=_gpu_like(64, 2, 128), v_pool=_gpu_like(64, 2, 128),
                cu_seqlens_q=i32(3), block_table=i32(2, 4), kv_lens=i32(2), max_seqlen_q=2,
                cu_rows=i32(2), prefix_lens=i32(1))
    for bad in (dict(q=_gpu_like(3, 12, 64)), dict(q=_gpu_like(3, 12, 128, dtype=torch.float32)),
                dict(q=_gpu_like(3, 5, 128)), dict(k_pool=_gpu_like(48, 2, 128)),
                dict(k_pool=_gpu_like(64, 2, 128, dtype=torch.float16)), dict(cu_seqlens_q=i32(4)),
                dict(kv_lens=torch.zeros(2)), dict(kv_lens=i32(4)[::2]), dict(prefix_lens=i32(2)),
                dict(cu_rows=i32(4), prefix_lens=i32(3)), dict(block_table=i32(3, 4)),
                dict(block_table=i32(2, 8)[:, ::2]), dict(block_size=24), dict(max_kv_len=65),
                dict(max_kv_len=-1), dict(max_seqlen_q=-1), dict(out=_gpu_like(3, 12, 64)),
                dict(out=_gpu_like(3, 12, 128, dtype=torch.float16))):
        with pytest.raises(AssertionError):
            shared.fa2_paged_shared(**{**good, **bad})
