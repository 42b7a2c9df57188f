"""Attention of new tokens over a paged cache whose rows share blocks, on the HIP kernel
(csrc/shared_attn.hip, through libmi_cache.so, the C ABI in include/mi_cache.h).

`fa2_paged_shared` is `fa2_paged_varlen` for a step some of whose rows are branches of one history
(KVCache.fork): it takes the groups of rows that share blocks and reads the shared ones once for
a group's rows, where the reference (and fa2_paged, fa2_paged_varlen) reads every row's keys for
that row alone (model.py:97,103).  No CPU path: CPU tensors are rejected.
"""
import math

import torch

from . import _lib
from .blocks import check, load
from .fa2 import HEAD_DIM, _dims_ok, _envelope, _strides, fa2_paged_varlen

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
                 sees them.
    is_causal    bottom-right aligned per row (query i of row b sees keys <= i + kv_len - T_b)
    out          optional [total_q, Hq, 128] output (any token/head strides); tokens of no row keep
                 what they hold
    More than 512 rows go to fa2_paged_varlen, which reads every row's keys for that row alone.
    Returns O [total_q, Hq, 128] (and the fp32 LSE [Hq, total_q] if return_lse).
    """
    assert q.is_cuda and k_pool.is_cuda and v_pool.is_cuda, "q and the pools must be GPU tensors"
    assert q.dim() == 3, "q is [total_q, Hq, d]"
    total_q, Hq, d = q.shape
    B = cu_seqlens_q.shape[0] - 1
    assert k_pool.dim() == 3 and k_pool.shape == v_pool.shape, "pools are [slots, Hkv, d]"
    assert k_pool.stride() == v_pool.stride(), "k_pool and v_pool must share strides"
    Hkv = k_pool.shape[1]
    assert Hq % Hkv == 0, "query heads must be a multiple of kv heads (GQA)"
    dev = q.device
    for t, name, shape in ((cu_seqlens_q, "cu_seqlens_q", (B + 1,)), (kv_lens, "kv_lens", (B,)),
                           (prefix_lens, "prefix_lens", (cu_rows.shape[0] - 1,)),
                           (cu_rows, "cu_rows", (prefix_lens.shape[0] + 1,))):
        assert t.dtype == torch.int32 and t.device == dev and t.shape == shape, \
            f"{name}: int32 of shape {shape} on {dev}"
        assert t.shape[0] <= 1 or t.stride(0) == 1, f"{name} must be contiguous"
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == B
    assert block_table.device == dev and k_pool.device == dev and v_pool.device == dev, \
        f"the pools and the table must be on {dev}"
    assert block_table.stride(-1) == 1 or block_table.shape[1] <= 1, \
        "block_table rows must be contiguous"
    assert prefix_lens.shape[0] <= B, "at most as many groups as rows"
    assert block_size >= 16 and block_size & (block_size - 1) == 0, "block_size: power of 2, >= 16"
    assert k_pool.shape[0] % block_size == 0, "pool slots must be whole blocks"
    _envelope(q, k_pool, v_pool)
    if max_kv_len is None:
        max_kv_len = block_table.shape[1] * block_size
    assert 0 <= max_kv_len <= block_table.shape[1] * block_size, \
        "max_kv_len exceeds what the block table can address"
    assert 0 <= max_seqlen_q, "max_seqlen_q must not be negative"
    if B > MAX_ROWS:
        return fa2_paged_varlen(q, k_pool, v_pool, cu_seqlens_q, block_table, kv_lens, max_seqlen_q,
                                block_size=block_size, max_kv_len=max_kv_len, is_causal=is_causal,
                                out=out, return_lse=return_lse)
    if not _dims_ok(q):
        q = q.clone(memory_format=torch.contiguous_format)   # 16-byte vector loads
    assert _dims_ok(k_pool) and _dims_ok(v_pool), "pools need 16-byte aligned token rows"
    O = out if out is not None else torch.empty((total_q, Hq, d), device=dev, dtype=q.dtype)
    assert O.shape == q.shape and O.dtype == q.dtype and O.device == dev and _dims_ok(O)
    L = torch.empty((Hq, total_q), device=dev, dtype=torch.float32) if return_lse else None
    lib = load()
    # every call has its own (from torch's caching allocator, in stream order): nothing is shared
    ws = torch.empty(lib.mi_cache_attend_workspace_size(total_q, Hq), dtype=torch.uint8, device=dev)
    with _lib.on_device(dev) as stream:
        check(lib.mi_cache_attend(
            _lib.DTYPES[q.dtype], q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), O.data_ptr(),
            L.data_ptr() if L is not None else None, cu_seqlens_q.data_ptr(),
            block_table.data_ptr(), block_table.stride(0) if B > 1 else block_table.shape[1],
            kv_lens.data_ptr(), cu_rows.data_ptr(), prefix_lens.data_ptr(), prefix_lens.shape[0], B,
            total_q, Hq, Hkv, int(max_kv_len), d, block_size, k_pool.shape[0] // block_size,
            _strides(q), _strides(k_pool), _strides(O),
            _strides(L) if L is not None else None, int(bool(is_causal)), 1.0 / math.sqrt(HEAD_DIM),
            ws.data_ptr(), ws.numel(), stream))
    return (O, L) if return_lse else O
