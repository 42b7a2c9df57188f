"""Blocks of a paged cache copied, forked and moved together on the HIP kernels (csrc/block_ops.hip,
through libmi_cache.so, the C ABI in include/mi_cache.h).

  copy_blocks   blocks of one pool into another (or the same)
  fork_rows     new sequences over another's history: whole blocks shared, the started one copied
  move_blocks   blocks moved, and the tables that name them rewritten

The reference's cache has none of them: every sequence owns all its blocks (kv_cache.py:31-72).  A
pool is KVCache.buf, [layers, 2, slots, kv_heads, d] (or any [..., slots, kv_heads, d] whose blocks
are contiguous); each call is one launch over all its planes.  KVCache.fork, copy_from and compact
keep the books around them.  No CPU path: CPU tensors are rejected.
"""
import ctypes
import os
from pathlib import Path

import torch

from . import _lib
from .fa2 import _MEMO_MAX

LIB_PATH = Path(os.environ.get("MI_CACHE_LIB", Path(__file__).resolve().parent / "libmi_cache.so"))

_p, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
_sz = ctypes.c_size_t
# name -> (restype, argtypes); mirrors include/mi_cache.h
SIGNATURES = {
    "mi_cache_last_error": (ctypes.c_char_p, []),
    "mi_cache_copy_blocks": (_i32, [_p, _i64, _i32, _p, _i64, _i32, _i32, _i64, _p, _i32, _p]),
    "mi_cache_fork_rows": (_i32, [_p, _i64, _i32, _i32, _i32, _i64, _p, _i64, _i32, _p, _i32, _p,
                                  _i32, _p]),
    "mi_cache_move_blocks": (_i32, [_p, _i64, _i32, _i32, _i64, _p, _i32, _p, _i64, _i32, _i32, _p,
                                    _i32, _p, _p]),
    "mi_cache_attend_workspace_size": (_sz, [_i32, _i32]),
    "mi_cache_attend": (_i32, [_i32, _p, _p, _p, _p, _p, _p, _p, _i64, _p, _p, _p, _i32, _i32, _i32,
                               _i32, _i32, _i32, _i32, _i32, _i32, _p, _p, _p, _p, _i32, _f32, _p,
                               _sz, _p]),
}

_library = None


def load():
    """Load libmi_cache.so once; raise if it is missing."""
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
        raise _lib.MiFa2Error(
            f"libmi_cache status {status}: {load().mi_cache_last_error().decode()}")


_PLANS = {}   # per entry point and its arguments' shapes, strides, types and devices: what to launch


def _plan(key, make, *args):
    """make(*args), which runs every check that those decide, once per combination."""
    if len(_PLANS) >= _MEMO_MAX:
        _PLANS.clear()
    got = _PLANS[key] = make(*args)
    return got


def call(device, fn, *args):
    """fn(*args, stream) on the device's current stream; raises what it reports."""
    if device == torch._C._cuda_getDevice():
        check(fn(*args, torch._C._cuda_getCurrentRawStream(device)))
        return
    with _lib.on_device(torch.device("cuda", device)) as stream:
        check(fn(*args, stream))


def _planes(pool, name, block_size):
    """(planes, bytes between them, blocks, bytes of a block) of a pool [..., slots, kv_heads, d]."""
    assert pool.is_cuda, f"{name}: a GPU tensor"
    assert pool.dim() >= 3, f"{name}: [..., slots, kv_heads, d]"
    slots, heads, d = pool.shape[-3:]
    assert type(block_size) is int and block_size > 0, "block_size: a positive int"
    assert slots % block_size == 0, f"{name}: slots must be whole blocks"
    # a block is one run of memory: strides of dimensions of one entry say nothing
    run = 1
    for size, stride in zip((d, heads, slots), reversed(pool.stride()[-3:])):
        assert size <= 1 or stride == run, f"{name}: the last three dimensions must be contiguous"
        run *= size
    planes, step = 1, run
    for size, stride in zip(reversed(pool.shape[:-3]), reversed(pool.stride()[:-3])):
        if size != 1:
            assert planes == 1 or stride == step * planes, f"{name}: planes must be evenly apart"
            if planes == 1:
                step = stride
            planes *= size
    assert planes == 1 or step >= run, f"{name}: planes must not overlap"
    n = pool.element_size()
    return planes, step * n, slots // block_size, block_size * heads * d * n


def _ids(t, name, shape, device):
    """A contiguous int32 tensor of that shape (its first entry None: any)."""
    got = t.shape
    assert (t.dtype == torch.int32 and len(got) == len(shape) and got[1:] == shape[1:]
            and shape[0] in (None, got[0]) and t.is_contiguous() and t.device == device), \
        f"{name}: contiguous int32 of shape {shape} on {device}"


def _table(tables, device):
    """(entries between rows, entries of a row, rows)."""
    assert tables.device == device and tables.dtype == torch.int32 and tables.dim() == 2, \
        f"tables: [max_seqs, width] int32 on {device}"
    assert tables.stride(1) == 1 or tables.shape[1] <= 1, "tables: rows must be contiguous"
    stride = tables.stride(0) if tables.shape[0] > 1 else tables.shape[1]
    return stride, tables.shape[1], tables.shape[0]


def _parts(n, planes, size, rows=0):
    """(first, count) of n blocks, a launch each: 2^23 work-groups of 16 KB at most."""
    most = max(1, ((1 << 23) - rows) // (planes * -(-size // 16384)) - 2)
    return [(i, min(n, i + most) - i) for i in range(0, max(n, 1), most)]


def copy_blocks(src_pool, dst_pool, pairs, block_size):
    """dst_pool's block pairs[i, 1] = src_pool's block pairs[i, 0], in every plane; returns dst_pool.

    pairs [n, 2] int32 on the pools' device.  The pools have the same planes, kv_heads, d and dtype,
    their own numbers of blocks, and may be one pool.  No block may be written twice, nor (in one
    pool) be both read and written.  Pairs outside the pools are skipped."""
    assert type(block_size) is int, "block_size: a positive int"   # (16.0 would find 16's plan)
    key = ("copy", block_size, src_pool.shape, src_pool.stride(), src_pool.dtype, src_pool.device,
           dst_pool.shape, dst_pool.stride(), dst_pool.dtype, dst_pool.device, pairs.shape,
           pairs.stride(), pairs.dtype, pairs.device)
    plan = _PLANS.get(key)
    if plan is None:
        plan = _plan(key, _copy_plan, src_pool, dst_pool, pairs, block_size)
    device, fn, src_step, src_blocks, dst, parts = plan
    for first, n in parts:
        call(device, fn, src_pool.data_ptr(), src_step, src_blocks, dst_pool.data_ptr(), *dst,
              pairs.data_ptr() + 8 * first, n)
    return dst_pool


def _copy_plan(src_pool, dst_pool, pairs, block_size):
    assert src_pool.dtype == dst_pool.dtype and src_pool.device == dst_pool.device, \
        "pools of one dtype on one device"
    assert src_pool.shape[:-3] == dst_pool.shape[:-3] and src_pool.shape[-2:] == dst_pool.shape[-2:], \
        "pools of the same planes, kv heads and head dim"
    planes, src_step, src_blocks, size = _planes(src_pool, "src_pool", block_size)
    _, dst_step, dst_blocks, _ = _planes(dst_pool, "dst_pool", block_size)
    _ids(pairs, "pairs", (None, 2), src_pool.device)
    nothing = size == 0 or planes == 0 or pairs.shape[0] == 0
    return (src_pool.device.index, load().mi_cache_copy_blocks, src_step, src_blocks,
            (dst_step, dst_blocks, planes, size), [] if nothing else _parts(pairs.shape[0], planes, size))


def fork_rows(pool, tables, lens, children, block_size):
    """New sequences over another's history, in place in `pool`, `tables` [max_seqs, width] int32 and
    `lens` [max_seqs] int32.

    children [n, 4] int32: parent slot, child slot, tokens L, new block.  The child's table begins
    with the parent's L // block_size whole blocks; the L % block_size tokens after them are copied
    into the new block (not looked at where there are none), which is its next entry; its length
    becomes L.  Child slots and new blocks must be distinct, and no child slot may be a parent slot.  A
    child that names anything out of range is skipped whole."""
    assert type(block_size) is int, "block_size: a positive int"
    key = ("fork", block_size, pool.shape, pool.stride(), pool.dtype, pool.device, tables.shape,
           tables.stride(), tables.dtype, tables.device, lens.shape, lens.stride(), lens.dtype,
           lens.device, children.shape, children.stride(), children.dtype, children.device)
    plan = _PLANS.get(key)
    if plan is None:
        plan = _plan(key, _fork_plan, pool, tables, lens, children, block_size)
    device, fn, shape, table, n_seqs, parts = plan
    for first, n in parts:
        call(device, fn, pool.data_ptr(), *shape, tables.data_ptr(), *table, lens.data_ptr(), n_seqs,
              children.data_ptr() + 16 * first, n)


def _fork_plan(pool, tables, lens, children, block_size):
    planes, step, blocks, size = _planes(pool, "pool", block_size)
    assert size and planes, "pool: no values"
    stride, width, n_seqs = _table(tables, pool.device)
    _ids(lens, "lens", (n_seqs,), pool.device)
    _ids(children, "children", (None, 4), pool.device)
    n = children.shape[0] if n_seqs else 0
    return (pool.device.index, load().mi_cache_fork_rows,
            (step, blocks, planes, block_size, size // block_size), (stride, width), n_seqs,
            _parts(n, planes, size, n) if n else [])


def move_blocks(pool, tables, rows, pairs, new_ids, block_size):
    """Block pairs[i, 1] = block pairs[i, 0] in every plane of `pool`, and the tables that name moved
    blocks rewritten: tables[slot, j] = new_ids[tables[slot, j]] for j < held, (slot, held) = rows[i].

    pairs [n, 2], rows [n_rows, 2], new_ids [blocks of the pool] int32 (a block that stays has its own
    id).  No block may be both read and written or written twice, and no slot may occur twice."""
    assert type(block_size) is int, "block_size: a positive int"
    key = ("move", block_size, pool.shape, pool.stride(), pool.dtype, pool.device, tables.shape,
           tables.stride(), tables.dtype, tables.device, rows.shape, rows.stride(), rows.dtype,
           rows.device, pairs.shape, pairs.stride(), pairs.dtype, pairs.device, new_ids.shape,
           new_ids.stride(), new_ids.dtype, new_ids.device)
    plan = _PLANS.get(key)
    if plan is None:
        plan = _plan(key, _move_plan, pool, tables, rows, pairs, new_ids, block_size)
    device, fn, shape, table, n_rows, parts = plan
    for first, n in parts:
        call(device, fn, pool.data_ptr(), *shape, pairs.data_ptr() + 8 * first, n, tables.data_ptr(),
              *table, rows.data_ptr(), 0 if first else n_rows, new_ids.data_ptr())


def _move_plan(pool, tables, rows, pairs, new_ids, block_size):
    planes, step, blocks, size = _planes(pool, "pool", block_size)
    assert size and planes, "pool: no values"
    table = _table(tables, pool.device)
    _ids(pairs, "pairs", (None, 2), pool.device)
    _ids(rows, "rows", (None, 2), pool.device)
    _ids(new_ids, "new_ids", (blocks,), pool.device)
    n, n_rows = pairs.shape[0], rows.shape[0]
    return (pool.device.index, load().mi_cache_move_blocks, (step, blocks, planes, size),
            table, n_rows, _parts(n, planes, size, n_rows) if n or n_rows else [])
