"""Attention over shared blocks (csrc/shared_attn.hip) against the definition in 64 bits.

The bound on a value.  The weights p of a query are rounded to the 16-bit type (half a step: relative
u) and summed as rounded; they are exact otherwise up to fp32.  With w = p / sum p,
|o' - o| <= u sum w |v - o| / (1 - u) <= u (A + |o|) / (1 - u), A = sum w |v|, and rounding o' adds
u |o'|: u (A + 2 |o|) to first order, held to 1.02 times that.  In fp16 a p below 2^-14 is off by up to
2^-25, the sum being at least 1: another S 2^-25 max |v|.  Scores, exponentials, sums and the merge
of key ranges are fp32: for scores of magnitude s (in bits) exp2 is off by s 2^-23 and a sum of 128
products by 2^-20 of their magnitudes, below 2^-12 A for the values here (|s| < 200).
"""
import math
import random

import pytest
import torch

from conftest import announce
from kernels.shared import fa2_paged_shared

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Batch:
    """Rows over a pool of blocks: groups [(rows, prefix tokens shared by blocks)], own[b] tokens behind
    them, new[b] queries.  Everything not held by a row is NaN."""

    def __init__(self, groups, own, new, *, heads=(12, 2), bs=16, dtype="bf16", seed=0, q_scale=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = random.Random(seed)
        self.bs, self.heads, dt = bs, heads, DT[dtype]
        self.dtype, self.new = dt, new
        tables, n, self.kv, sizes, prefix = [], 0, [], [], []
        for size, p in groups:
            assert p % bs == 0
            shared = list(range(n, n + p // bs))
            n += len(shared)
            for _ in range(size):
                b = len(tables)
                mine = -(-own[b] // bs)
                tables.append(shared + list(range(n, n + mine)))
                n += mine
                self.kv.append(p + own[b])
            sizes.append(size)
            prefix.append(p)
        ids = r.sample(range(n + 3), n + 3)
        self.tables = [[ids[x] for x in t] for t in tables]
        width = max(1, max(map(len, tables)) + 2)
        # entries past a row's blocks: anything
        self.table = i32([t + [r.choice([-5, n + 3, 2**31 - 1])] * (width - len(t))
                          for t in self.tables])
        self.pool = torch.full((2, (n + 3) * bs, heads[1], 128), math.nan, dtype=dt, device="cuda")
        for t, kv in zip(self.tables, self.kv):
            slots = self.slots(t, kv)
            hole = self.pool[0, slots, 0, 0].isnan()
            self.pool[:, slots[hole]] = torch.randn(2, int(hole.sum()), heads[1], 128, generator=g,
                                                    device="cuda").to(dt)
        cu = [0]
        for c in new:
            cu.append(cu[-1] + c)
        self.cu = cu
        self.q = (torch.randn(cu[-1], heads[0], 128, generator=g, device="cuda") * q_scale).to(dt)
        rows = [0]
        for s in sizes:
            rows.append(rows[-1] + s)
        self.cu_rows, self.prefix, self.lens = i32(rows), i32(prefix), i32(self.kv)
        self.cu_q = i32(cu)

    def slots(self, table, n):
        t = torch.tensor(table[:-(-n // self.bs)], dtype=torch.long, device="cuda")
        return (t[:, None] * self.bs + torch.arange(self.bs, device="cuda")).reshape(-1)[:n]

    def call(self, **over):
        a = dict(q=self.q, k_pool=self.pool[0], v_pool=self.pool[1], cu_seqlens_q=self.cu_q,
                 block_table=self.table, kv_lens=self.lens, max_seqlen_q=max(self.new, default=0),
                 cu_rows=self.cu_rows, prefix_lens=self.prefix, block_size=self.bs,
                 max_kv_len=max(self.kv))
        a.update(over)
        return fa2_paged_shared(**a)

    def exact(self, causal=True):
        """(o, sum w |v|, lse) in 64 bits."""
        Hq, Hkv = self.heads
        o = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        A = torch.zeros_like(o)
        lse = torch.full((Hq, o.shape[0]), -math.inf, dtype=torch.float64, device="cuda")
        for b, (t, n) in enumerate(zip(self.tables, self.kv)):
            lo, hi = self.cu[b], self.cu[b + 1]
            if lo == hi or n == 0:
                continue
            s = self.slots(t, n)
            k = self.pool[0, s].double().repeat_interleave(Hq // Hkv, 1).transpose(0, 1)
            v = self.pool[1, s].double().repeat_interleave(Hq // Hkv, 1).transpose(0, 1)
            q = self.q[lo:hi].double().transpose(0, 1)
            sc = (q @ k.transpose(1, 2).contiguous()) / math.sqrt(128)
            if causal:
                at = torch.arange(n, device="cuda")[None, :]
                sc.masked_fill_(at > torch.arange(hi - lo, device="cuda")[:, None] + n - (hi - lo),
                                -math.inf)
            w = torch.nan_to_num(torch.softmax(sc, -1))
            o[lo:hi] = (w @ v).transpose(0, 1)
            A[lo:hi] = (w @ v.abs()).transpose(0, 1)
            lse[:, lo:hi] = torch.logsumexp(sc, -1)
        return o, A, lse

    def bound(self, o, A):
        u = torch.finfo(self.dtype).eps / 2
        bound = 1.02 * u * (A + 2 * o.abs()) + 2.0 ** -12 * A
        if self.dtype == torch.float16:
            bound += max(self.kv) * 2.0 ** -25 * 6 + 2.0 ** -25
        return bound

    def check(self, out, lse=None, causal=True):
        o, A, want = self.exact(causal)
        bound = self.bound(o, A)
        u = torch.finfo(self.dtype).eps / 2
        err = (out.double() - o).abs()
        assert not out.isnan().any()
        worst = err / bound.clamp_min(1e-30)
        assert worst.max() <= 1, f"{worst.max().item():.3f} of the bound at {worst.argmax().item()}"
        if lse is not None:
            seen = want.isfinite()
            assert torch.equal(lse.isfinite(), seen) and (lse[~seen] == -math.inf).all()
            # sums of rounded weights: relative u; scores fp32
            off = (lse.double() - want)[seen].abs()
            assert (off <= 1.02 * u + 1e-4 + want[seen].abs() * 1e-6).all(), off.max().item()


def rand(r, lo, hi):
    return round(math.exp(r.uniform(math.log(lo), math.log(hi))))


CASES = [
    # groups (rows, prefix), own tokens, new tokens
    dict(groups=[(2, 96)], own=[5, 9], new=[1, 1]),
    dict(groups=[(1, 0)], own=[1], new=[1]),
    dict(groups=[(1, 16)], own=[1], new=[1]),
    dict(groups=[(3, 16)], own=[1, 16, 17], new=[1, 1, 1]),
    dict(groups=[(16, 2048)], own=list(range(1, 17)), new=[1] * 16),
    dict(groups=[(5, 48), (1, 0), (1, 512), (4, 160), (2, 0)],
         own=[1, 300, 31, 32, 33, 700, 2, 5, 16, 129, 128, 64, 1], new=[1] * 13),
    dict(groups=[(64, 304)], own=[1 + (7 * i) % 90 for i in range(64)], new=[1] * 64),
    # chunks, ragged, with rows without queries
    dict(groups=[(4, 128)], own=[20, 7, 33, 1], new=[5, 7, 0, 1]),
    dict(groups=[(3, 640), (2, 32)], own=[64, 65, 63, 200, 10], new=[64, 17, 33, 2, 3]),
    dict(groups=[(2, 400)], own=[150, 333], new=[150, 90]),
    # more queries than keys: the first see nothing; a row without keys
    dict(groups=[(1, 0), (1, 0), (2, 0)], own=[3, 0, 1, 8], new=[8, 4, 2, 8]),
    dict(groups=[(2, 16)], own=[2, 5], new=[20, 3]),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_shapes(i, dtype):
    announce(f"shared attention case {i} {dtype}")
    b = Batch(**CASES[i], dtype=dtype, seed=i)
    out, lse = b.call(return_lse=True)
    b.check(out, lse)
    assert torch.equal(out, b.call())                 # without the lse, and again
    out, lse = b.call(is_causal=False, return_lse=True)
    b.check(out, lse, causal=False)


@pytest.mark.parametrize("heads", [(8, 8), (5, 1), (32, 8), (14, 2), (16, 1), (17, 1), (40, 1), (3, 3)])
@pytest.mark.parametrize("bs", [16, 64, 512])
def test_head_layouts_and_block_sizes(heads, bs):
    announce(f"shared attention heads {heads} blocks of {bs}")
    b = Batch([(3, 2 * bs), (2, bs), (1, 0)], [1, 40, bs + 3, 9, 2 * bs, 77], [1, 3, 2, 1, 7, 5],
              heads=heads, bs=bs, seed=bs)
    out, lse = b.call(return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("seed", range(24))
def test_drawn(seed):
    r = random.Random(seed)
    n_groups, bs = r.randint(1, 7), r.choice([16, 16, 32, 128])
    groups = [(r.randint(1, 9), rand(r, 1, 3000) // bs * bs) for _ in range(n_groups)]
    rows = sum(s for s, _ in groups)
    most = r.choice([1, 1, rand(r, 1, 100)])
    new = [r.randint(0 if most > 1 else 1, most) for _ in range(rows)]
    own = [max(n, rand(r, 1, 600)) for n in new]
    heads = r.choice([(12, 2), (12, 2), (8, 2), (4, 4), (6, 1)])
    announce(f"shared attention drawn {seed}: {groups} {heads} {bs} most {most}")
    b = Batch(groups, own, new, heads=heads, bs=bs, dtype=r.choice(["bf16", "fp16"]), seed=seed)
    out, lse = b.call(return_lse=True)
    b.check(out, lse)


def test_groups_as_they_come():
    # whatever the groups say of rows that hold the same tokens, the result is the same attention
    b = Batch([(4, 320)], [7, 30, 1, 64], [1, 4, 1, 2], seed=5)
    want = b.call()
    b.check(want)
    for rows, prefix in [([0, 4], [17]), ([0, 4], [100000]), ([0, 4], [-3]), ([0, 1, 2, 3, 4], [320] * 4),
                         ([0, 0, 3, 3, 4], [9, 320, 5, 320]), ([1, 3], [300]), ([0], []),
                         ([0, 2, 4], [320, 64]), ([0, 3, 4, 4, 4], [320, 0, 320, 320]),
                         ([-5, 2], [320]), ([2, 9], [320]), ([3, 1], [320]), ([0, 4, 0, 4], [320, 1, 64])]:
        b.check(b.call(cu_rows=i32(rows), prefix_lens=i32(prefix)))


def test_first_row_shorter_than_the_prefix():
    # the group's first row holds less than the prefix (a padding row holds nothing): what it does not
    # hold is read through the rows' own tables
    b = Batch([(4, 320)], [7, 30, 1, 64], [1, 4, 1, 2], seed=6)
    table = b.table.clone()
    for short in (0, 5, 100):
        b.table = table.clone()
        for row in (0, 2):
            b.kv[row] = short
            b.lens = i32(b.kv)
            if short == 0:
                b.table[row] = 2**31 - 1
            b.check(b.call())


def test_lengths_clamped_to_the_bound():
    b = Batch([(2, 64)], [100, 30], [1, 2], seed=7)
    full = b.lens.clone()
    b.kv = [90, 90]
    b.lens = i32(b.kv)
    want = b.call(max_kv_len=90)
    assert torch.equal(b.call(kv_lens=full, max_kv_len=90), want)
    b.check(want)
    assert not b.call(kv_lens=i32([-4, 0])).any()
    assert not b.call(max_kv_len=0).any()


def test_tokens_of_no_row_keep_what_they_hold():
    b = Batch([(2, 64)], [10, 30], [2, 3], seed=8)
    want = b.call()
    q = torch.cat([torch.full_like(b.q[:4], math.nan), b.q, torch.full_like(b.q[:3], math.nan)])
    out = torch.full_like(q, 7.0)
    got = b.call(q=q, cu_seqlens_q=b.cu_q + 4, out=out)
    assert got is out and torch.equal(out[4:9], want)
    assert (out[:4] == 7).all() and (out[9:] == 7).all()


def test_strides():
    b = Batch([(3, 128)], [10, 30, 5], [2, 3, 1], heads=(6, 2), seed=9)
    want = b.call()
    wide = torch.full((b.q.shape[0], 9, 160), math.nan, dtype=b.dtype, device="cuda")
    wide[:, 1:7, 16:144] = b.q
    out = torch.full((6, b.q.shape[0], 136), 3.0, dtype=b.dtype, device="cuda")
    got = b.call(q=wide[:, 1:7, 16:144], out=out.transpose(0, 1)[..., :128])
    assert torch.equal(got, want) and (out[..., 128:] == 3).all()
    assert torch.equal(b.call(q=wide[:, 1:7, 16:144].transpose(0, 1).contiguous().transpose(0, 1)), want)
    odd = torch.empty(b.q.numel() + 3, dtype=b.dtype, device="cuda")[3:].view(b.q.shape)
    odd.copy_(b.q)                                   # not 16-byte aligned
    assert torch.equal(b.call(q=odd), want)
    # pools inside a whole cache's buffer with more heads per slot
    both = torch.full((b.pool.shape[1], 2, 3, 128), math.nan, dtype=b.dtype, device="cuda")
    both[:, :, :2] = b.pool.transpose(0, 1)
    assert torch.equal(b.call(k_pool=both[:, 0, :2], v_pool=both[:, 1, :2]), want)


def test_one_table_for_all_rows():
    # an expanded table: every row the same sequence at another length
    b = Batch([(1, 0)], [300], [1], seed=10)
    b.new, b.cu = [1, 1, 1], [0, 1, 2, 3]
    b.q = torch.randn(3, 12, 128, device="cuda").to(b.dtype)
    b.tables, b.kv = b.tables * 3, [300, 7, 256]
    b.check(b.call(q=b.q, cu_seqlens_q=i32(b.cu), block_table=b.table.expand(3, -1),
                   kv_lens=i32(b.kv), cu_rows=i32([0, 3]), prefix_lens=i32([250])))


def test_large_scores():
    # scores up to some 10^3 in bits, where one key takes all the weight; ties between equal keys
    b = Batch([(3, 512)], [40, 3, 70], [1, 2, 1], seed=11)
    big = b.q * 64
    b.q = big.to(b.dtype)
    out = b.call()
    o, _, _ = b.exact()
    # |v| and so A and |o| are at most 5; the products of a score sum to some 700 in magnitude (in
    # bits), 128 of them in fp32 to 128 * 2^-24 * 700 < 2^-7: weights are off by as much, twice
    assert ((out.double() - o).abs() <= 2.0 ** -8 * 1.02 * 15 + 5 * 2.0 ** -6).all()
    b.pool[0, :] = torch.where(b.pool[0].isnan(), b.pool[0], torch.ones_like(b.pool[0]))
    for q in (2.0 ** 20, 2.0 ** 60):   # equal scores of some 2^24 and 2^64: equal weights
        b.q = torch.full_like(b.q, q)
        b.check(b.call())


def test_values_behind_the_mask():
    # a later new token's value may be inf or NaN: an earlier query does not see it
    b = Batch([(2, 64)], [40, 33], [6, 3], seed=12)
    o, A, _ = b.exact()
    for row, last in enumerate(b.kv):
        slot = int(b.slots(b.tables[row], last)[-1])
        b.pool[1, slot] = math.nan if row else math.inf
        b.pool[0, slot] = math.nan
    got = b.call()
    for lo, hi in zip(b.cu[:-1], b.cu[1:]):
        at = slice(lo, hi - 1)
        assert ((got[at].double() - o[at]).abs() <= b.bound(o[at], A[at])).all()
        assert got[hi - 1].isnan().all()


def test_on_a_side_stream_and_in_graphs():
    b = Batch([(6, 320), (1, 0)], [5, 60, 17, 1, 100, 33, 40], [1] * 7, seed=13)
    want = b.call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = b.call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    # two graphs of one stream, lengths and groups changed between replays
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = b.call(max_kv_len=b.table.shape[1] * b.bs)
        graphs.append((graph, out))
    for kv, rows, prefix in [(b.kv, [0, 6, 7], [320, 0]), ([n - 1 for n in b.kv], [0, 6, 7], [304, 0]),
                             ([n // 2 for n in b.kv], [0, 7, 7], [0, 0]), (b.kv, [0, 6, 7], [320, 0])]:
        b.kv = kv
        b.lens.copy_(i32(kv))
        b.cu_rows.copy_(i32(rows))
        b.prefix.copy_(i32(prefix))
        torch.cuda.synchronize()
        eager = b.call(max_kv_len=b.table.shape[1] * b.bs)
        for graph, out in graphs:
            graph.replay()
        for graph, out in graphs:
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
            graph.replay()
        b.check(eager)


def test_long_cache_offsets_past_32_bits():
    # a pool of 5 GB, the rows' blocks at its far end
    bs, heads = 64, (8, 8)
    slots = (5 << 30) // (8 * 128 * 2) // bs * bs
    b = Batch([(3, 256)], [10, 70, 64], [1, 2, 1], heads=heads, bs=bs, seed=14)
    want = b.call()
    far = torch.zeros(2, slots, 8, 128, dtype=b.dtype, device="cuda")
    n = b.pool.shape[1]
    far[:, slots - n:] = b.pool
    held = b.table.clone()
    b.table = torch.where((held >= 0) & (held < n // bs), held + (slots - n) // bs, held)
    assert torch.equal(b.call(k_pool=far[0], v_pool=far[1], block_table=b.table.contiguous()), want)


@pytest.mark.parametrize("rows", [512, 513, 1024])
def test_many_rows(rows):
    # 512 on the kernel, more on fa2_paged_varlen
    b = Batch([(rows - 24, 64), (24, 32)], [1 + i % 5 for i in range(rows)], [1] * rows, heads=(4, 2),
              seed=15)
    out, lse = b.call(return_lse=True)
    b.check(out, lse)


def test_nothing_to_do():
    b = Batch([(2, 32)], [3, 4], [0, 0], seed=16)
    assert b.call().shape == (0, 12, 128)
    empty = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    out = fa2_paged_shared(b.q, b.pool[0], b.pool[1], i32([0]), empty, i32([]), 0, i32([0]), i32([]))
    assert out.shape == (0, 12, 128)
