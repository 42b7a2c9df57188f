"""Attention over shared blocks (csrc/shared_attn.hip) where values are NaN or inf in places that a query
sees, and over key ranges long enough that a worker refills what it knows of their blocks.

A score that is NaN, or a value that is, makes the query's output NaN, whichever part of its keys it lies in
(the prefix, its own keys, one worker's share of either) and whatever that part weighs; the other
queries and heads keep their values.  Bounds as in test_shared_attn_gpu.py."""
import math

import pytest
import torch

from conftest import announce
from kernels.fa2 import fa2_paged
from test_shared_attn_gpu import DT, Batch

pytestmark = pytest.mark.gpu


def check(b, out, lse, odd):
    """NaN exactly where odd [tokens, heads] says, everything else as in 64 bits."""
    kept = b.q
    b.q = torch.where(kept.isnan(), torch.zeros_like(kept), kept)
    o, A, want = b.exact()
    b.q = kept
    assert torch.equal(out.isnan().all(-1), odd) and torch.equal(out.isnan().any(-1), odd)
    assert torch.equal(lse.isnan(), odd.t())
    ok = ~odd
    assert ((out.double() - o).abs()[ok] <= b.bound(o, A)[ok]).all()
    seen = want.isfinite() & ok.t()
    assert torch.equal(lse.isfinite(), seen)
    u = torch.finfo(b.dtype).eps / 2
    assert ((lse.double() - want)[seen].abs() <= 1.02 * u + 1e-4 + want[seen].abs() * 1e-6).all()


def nothing(b):
    return torch.zeros(b.q.shape[:2], dtype=torch.bool, device="cuda")


# The prefix pays to be read once in each: 18 pairs (a narrow range), 120 (one wide tile) and 1,080 (nine).
# Below 2,048 (token, head) pairs in all, four waves merge the parts of one, from there on half a wave.
SIZES = {"narrow": dict(groups=[(3, 320), (1, 0)], own=[5, 17, 40, 70], new=[1] * 4),
         "wide": dict(groups=[(20, 640), (1, 0)], own=[9 + 5 * i for i in range(21)], new=[1] * 21),
         "many": dict(groups=[(60, 2048), (1, 0)], own=[9 + 5 * i for i in range(61)], new=[3] * 61)}


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("size", SIZES)
def test_nan_queries(size, dtype):
    announce(f"shared attention, NaN queries, {size} {dtype}")
    b = Batch(**SIZES[size], dtype=dtype, seed=20)
    odd = nothing(b)
    for token, head in ((0, 0), (1, 7), (b.q.shape[0] - 1, 11)):
        b.q[token, head, 5] = math.nan
        odd[token, head] = True
    assert (odd.numel() >= 2048) == (size == "many")
    out, lse = b.call(return_lse=True)
    check(b, out, lse, odd)


@pytest.mark.parametrize("size", SIZES)
def test_a_nan_key_alone_in_its_part(size):
    # row 1's own range is one key, its new token's, with a NaN K in kv head 1: as it is when the last token
    # filled a block
    announce(f"shared attention, a NaN key alone, {size}")
    shape = {**SIZES[size], "own": [1 if i == 1 else n for i, n in enumerate(SIZES[size]["own"])],
             "new": [1 if i == 1 else n for i, n in enumerate(SIZES[size]["new"])]}
    b = Batch(**shape, seed=21)
    slot = b.slots(b.tables[1], b.kv[1])[-1:]
    b.pool[0, slot, 1, 3] = math.nan
    odd = nothing(b)
    odd[b.cu[1]:b.cu[2], 6:] = True
    out, lse = b.call(return_lse=True)
    check(b, out, lse, odd)
    if size == "narrow":     # the framework's attention of one row at a time agrees
        alone = fa2_paged(b.q.unsqueeze(2), b.pool[0], b.pool[1], b.table, b.lens, block_size=b.bs,
                          max_kv_len=max(b.kv))[:, :, 0]
        assert torch.equal(alone.isnan(), out.isnan())


def test_nan_keys_in_a_whole_prefix():
    # every key that the group shares, in one head: every part of it is NaN
    b = Batch([(6, 1600), (2, 0)], [5, 6, 7, 8, 9, 10, 30, 40], [1] * 8, seed=22)
    b.pool[0, b.slots(b.tables[0], 1600), 0] = math.nan
    odd = nothing(b)
    odd[:6, :6] = True
    out, lse = b.call(return_lse=True)
    check(b, out, lse, odd)


@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_odd_values_in_a_part_that_weighs_nothing(what, value):
    """One own key outweighs all others by some 700 bits, so that the prefix's part has no weight left in
    32 bits: a NaN there still shows, and so does an infinite score (inf - inf)."""
    b = Batch([(4, 320)], [20, 21, 22, 23], [1] * 4, seed=23)
    b.q[:] = 40.0
    for row in (1, 2):
        b.pool[0, b.slots(b.tables[row], b.kv[row])[-1]] = 1.5   # 1.5 * 40 * 128 / sqrt 128 = 679
    slot = b.slots(b.tables[0], 320)[100]
    b.pool[0 if what == "k" else 1, slot, 0, 64] = value
    out, lse = b.call(return_lse=True)
    if what == "k":       # every row sees the key: its score is NaN, or the infinite maximum
        assert out[:, :6].isnan().all() and not lse[:6].isfinite().any()
    else:                 # the value's dim alone
        assert not out[:, :6, 64].isfinite().any() and lse.isfinite().all()
        assert value == math.inf or out[:, :6, 64].isnan().all()
        assert out[:, :6, :64].isfinite().all() and out[:, :6, 65:].isfinite().all()
    assert out[:, 6:].isfinite().all() and lse[6:].isfinite().all()


def test_long_shares_of_wide_ranges():
    """A work-group that walks more than 64 steps of 128 keys finds the next 64 steps' blocks: 2,731 tokens of
    one row are 129 tiles of each kv head, 258 items of 97 steps each, about one for each work-group.

    Up to 97 * 64 products of a lane's stream are summed in fp32: off by 97 * 64 * 2^-24 < 2^-11 A."""
    announce("shared attention, wide shares of more than 64 steps")
    b = Batch([(1, 0)], [12300], [2731], seed=24)
    b.bound = lambda o, A: Batch.bound(b, o, A) + 2.0 ** -11 * A
    out, lse = b.call(return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_long_shares_of_narrow_ranges(dtype):
    """A wave that walks more than 16 units of 64 keys finds the next 32 steps' block ids: 64 rows of 36,000
    to 37,000 own keys, one kv head, are 36,000 units and more over at most 2,048 waves."""
    announce(f"shared attention, narrow shares of more than 16 units, {dtype}")
    g = torch.Generator(device="cuda").manual_seed(25)
    b = Batch([(2, 16)], [20, 30], [1, 1], heads=(4, 1), dtype=dtype, seed=25)
    kv = [36000 + 13 * i for i in range(64)]
    held = [-(-n // 16) for n in kv]
    ids = torch.randperm(sum(held), generator=torch.Generator().manual_seed(1)).tolist()
    b.tables, at = [], 0
    for n in held:
        b.tables.append(ids[at:at + n])
        at += n
    width = max(held)
    b.table = torch.tensor([t + [-1] * (width - len(t)) for t in b.tables], dtype=torch.int32,
                           device="cuda")
    b.kv, b.new, b.cu = kv, [1] * 64, list(range(65))
    b.pool = torch.randn(2, sum(held) * 16, 1, 128, generator=g, device="cuda").to(DT[dtype])
    b.q = torch.randn(64, 4, 128, generator=g, device="cuda").to(DT[dtype])
    b.lens, b.cu_q = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (kv, b.cu))
    b.cu_rows = torch.zeros(1, dtype=torch.int32, device="cuda")
    b.prefix = torch.zeros(0, dtype=torch.int32, device="cuda")
    out, lse = b.call(return_lse=True)
    b.check(out, lse)
