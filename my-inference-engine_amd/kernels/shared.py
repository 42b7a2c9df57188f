"""Attention of new tokens over a paged cache whose rows share blocks, on the HIP kernel
(csrc/shared_attn.hip, through libmi_cache.so, the C ABI in include/mi_cache.h).

`fa2_paged_shared` is `fa2_paged_varlen` for a step some of whose rows are branches of one history
(KVCache.fork): it takes the groups of rows that share blocks and reads the shared ones for all of
a group's rows together, where the reference (and fa2_paged, fa2_paged_varlen) reads every row's keys for
that row alone (model.py:97,103).  No CPU path: CPU tensors are rejected.
"""
import math
import operator

import torch

from . import _lib
from .blocks import call, load
from .fa2 import (_MEMO_MAX, HEAD_DIM, _contig, _dims_ok, _envelope, _strides, _strides_of,
                  _strides_ok, fa2_paged_varlen)

MAX_ROWS = 512   # rows of a call of the kernel


def fa2_paged_shared(q, k_pool, v_pool, cu_seqlens_q, block_table, kv_lens, max_seqlen_q, cu_rows,
                     prefix_lens, *, block_size=16, max_kv_len=None, is_causal=True, out=None,
                     return_lse=False):
    """Packed new tokens over the paged cache, the blocks that rows share read once for all of them.

    q            [total_q, Hq, 128]: row b's new queries are q[cu_q[b]:cu_q[b+1]] (rows may have
                 different counts, 0 included)
    k_pool/v_pool, block_table, kv_lens, block_size, max_kv_len: as in fa2_paged; kv_lens include
                 each row's new tokens, whose K/V are already in the pool
    max_seqlen_q host-side upper bound of the rows' counts
    cu_rows      [G + 1] int32, prefix_lens [G] int32, G <= rows: rows [cu_rows[g], cu_rows[g+1])
                 hold the same first prefix_lens[g] tokens (rows of no group share nothing).  They are
                 read through the table of the group's first row, as far as every query of the group
                 sees them and where that costs less than the rows by themselves.
    is_causal    bottom-right aligned per row (query i of row b sees keys <= i + kv_len - T_b)
    out          optional [total_q, Hq, 128] output (any token/head strides); tokens of no row keep
                 what they hold
    More than 512 rows go to fa2_paged_varlen, which reads every row's keys for that row alone.
    Worth it from tens of MB of K and V that the rows would read again (KVCache.sharing_pays has both
    sides' times).  Rows of more than a few tens of new tokens have full tiles of their own, and sharing saves
    them nothing: fa2_paged_varlen is faster (64 rows of up to 150 over 512 keys of 4 kv heads 66 us, here 107),
    but for few rows over long keys, which it does not cut (8 of 150 over 5,000 of 2 heads 73, here 54).
    Returns O [total_q, Hq, 128] (and the fp32 LSE [Hq, total_q] if return_lse).
    """
    # plain values only: the plan is looked up by them
    if type(max_kv_len) is not int and max_kv_len is not None:
        # the bound as given: rounding comes after
        assert 0 <= max_kv_len <= block_table.shape[1] * block_size, \
            "max_kv_len exceeds what the block table can address"
        max_kv_len = int(max_kv_len)
    assert 0 <= max_seqlen_q, "max_seqlen_q must not be negative"
    is_causal, return_lse = bool(is_causal), bool(return_lse)
    if type(block_size) is not int:
        block_size = operator.index(block_size)   # an integer of another type; a float is refused
    dev = q.device
    key = (q.shape, q.stride(), q.dtype, dev, k_pool.shape, k_pool.stride(), k_pool.dtype,
           k_pool.device, v_pool.shape, v_pool.stride(), v_pool.dtype, v_pool.device,
           cu_seqlens_q.shape, cu_seqlens_q.stride(), cu_seqlens_q.dtype, cu_seqlens_q.device,
           block_table.shape, block_table.stride(), block_table.dtype, block_table.device,
           kv_lens.shape, kv_lens.stride(), kv_lens.dtype, kv_lens.device, cu_rows.shape,
           cu_rows.stride(), cu_rows.dtype, cu_rows.device, prefix_lens.shape, prefix_lens.stride(),
           prefix_lens.dtype, prefix_lens.device, block_size, max_kv_len, is_causal, return_lse)
    pl = _PLANS.get(key)
    if pl is None:
        pl = _plan(q, k_pool, v_pool, cu_seqlens_q, block_table, kv_lens, cu_rows, prefix_lens,
                   block_size, max_kv_len, is_causal, return_lse)
        if len(_PLANS) >= _MEMO_MAX:
            _PLANS.clear()
        _PLANS[key] = pl
    (device, fn, dtype_code, many, copy_q, table_stride, sizes, q_st, pool_st, o_st, l_st, tail,
     ws_bytes) = pl
    kp, vp = k_pool.data_ptr(), v_pool.data_ptr()
    assert not (kp | vp) & 15, "pools need 16-byte aligned token rows"
    if many:
        return fa2_paged_varlen(q, k_pool, v_pool, cu_seqlens_q, block_table, kv_lens, max_seqlen_q,
                                block_size=block_size, max_kv_len=max_kv_len, is_causal=is_causal,
                                out=out, return_lse=return_lse)
    if copy_q or q.data_ptr() & 15:
        q = q.clone(memory_format=torch.contiguous_format)   # 16-byte vector loads
        q_st = _strides(q)
    if out is None:
        O = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        O = out
        assert O.shape == q.shape and O.dtype == q.dtype and O.device == dev and _dims_ok(O)
        o_st = _strides(O)
    L = torch.empty((q.shape[1], q.shape[0]), device=dev, dtype=torch.float32) if return_lse else None
    # every call has its own (from torch's caching allocator, in stream order): nothing is shared
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    call(device, fn, dtype_code, q.data_ptr(), kp, vp, O.data_ptr(), L.data_ptr() if return_lse else None,
         cu_seqlens_q.data_ptr(), block_table.data_ptr(), table_stride, kv_lens.data_ptr(),
         cu_rows.data_ptr(), prefix_lens.data_ptr(), *sizes, q_st, pool_st, o_st, l_st, *tail,
         ws.data_ptr(), ws_bytes)
    return (O, L) if return_lse else O


_PLANS = {}


def _plan(q, k_pool, v_pool, cu_seqlens_q, block_table, kv_lens, cu_rows, prefix_lens, block_size,
          max_kv_len, is_causal, return_lse):
    """Every check of fa2_paged_shared that its arguments' shapes, strides and types decide, then the
    launch's constant arguments (base alignment and `out` are checked per call)."""
    assert q.is_cuda and k_pool.is_cuda and v_pool.is_cuda, "q and the pools must be GPU tensors"
    assert q.dim() == 3, "q is [total_q, Hq, d]"
    total_q, Hq, d = q.shape
    B = cu_seqlens_q.shape[0] - 1
    assert k_pool.dim() == 3 and k_pool.shape == v_pool.shape, "pools are [slots, Hkv, d]"
    assert k_pool.stride() == v_pool.stride(), "k_pool and v_pool must share strides"
    Hkv = k_pool.shape[1]
    assert Hq % Hkv == 0, "query heads must be a multiple of kv heads (GQA)"
    dev, groups = q.device, prefix_lens.shape[0]
    for t, name, n in ((cu_seqlens_q, "cu_seqlens_q", B + 1), (kv_lens, "kv_lens", B),
                       (cu_rows, "cu_rows", groups + 1), (prefix_lens, "prefix_lens", groups)):
        assert t.dtype == torch.int32 and t.device == dev and t.shape == (n,), \
            f"{name}: {n} int32 on {dev}"
        assert n <= 1 or t.stride(0) == 1, f"{name} must be contiguous"
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == B
    assert block_table.device == dev and k_pool.device == dev and v_pool.device == dev, \
        f"the pools and the table must be on {dev}"
    width = block_table.shape[1]
    assert block_table.stride(-1) == 1 or width <= 1, "block_table rows must be contiguous"
    assert groups <= B, "at most as many groups as rows"
    assert block_size >= 16 and block_size & (block_size - 1) == 0, "block_size: power of 2, >= 16"
    assert k_pool.shape[0] % block_size == 0, "pool slots must be whole blocks"
    _envelope(q, k_pool, v_pool)
    if max_kv_len is None:
        max_kv_len = width * block_size
    # kv_lens are clamped to max_kv_len in-kernel, so this bound keeps every table read in range
    assert 0 <= max_kv_len <= width * block_size, \
        "max_kv_len exceeds what the block table can address"
    assert _strides_ok(k_pool) and _strides_ok(v_pool), "pools need 16-byte aligned token rows"
    return (dev.index, load().mi_cache_attend, _lib.DTYPES[q.dtype], B > MAX_ROWS, not _strides_ok(q),
            block_table.stride(0) if B > 1 else width,
            (groups, B, total_q, Hq, Hkv, max_kv_len, d, block_size, k_pool.shape[0] // block_size),
            _strides(q), _strides(k_pool), _strides_of(q.shape, _contig(q.shape)),
            _strides_of((Hq, total_q), (total_q, 1)) if return_lse else None,
            (int(is_causal), 1.0 / math.sqrt(HEAD_DIM)),
            load().mi_cache_attend_workspace_size(total_q, Hq))
