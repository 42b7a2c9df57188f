"""The block operations (csrc/block_ops.hip) against the same moves in torch indexing: every byte of
the pools, tables and lengths has to be equal."""
import random

import pytest
import torch

from conftest import announce
from kernels.blocks import copy_blocks, fork_rows, move_blocks

pytestmark = pytest.mark.gpu


def fill(*shape, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if dtype == torch.uint8:
        return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=dtype)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def i32(values, width=None):
    t = torch.tensor(values, dtype=torch.int32, device="cuda")
    return t.view(-1, width) if width else t


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# block sizes, heads and dims whose blocks are whole 16-byte words and ones that are not
SHAPES = [(2, 3, 2, 128, 16, torch.bfloat16), (1, 1, 8, 128, 128, torch.float16),
          (28, 2, 2, 128, 16, torch.bfloat16), (2, 2, 1, 64, 16, torch.float32),
          (1, 3, 3, 5, 1, torch.bfloat16), (2, 2, 1, 1, 3, torch.uint8), (1, 2, 4, 80, 32, torch.float16)]


@pytest.mark.parametrize("layers,planes,heads,d,bs,dtype", SHAPES)
@pytest.mark.parametrize("n", [1, 2, 13, 40])
def test_copy(layers, planes, heads, d, bs, dtype, n):
    announce(f"copy {layers}x{planes}x{heads}x{d} blocks of {bs} {dtype} n={n}")
    r = random.Random(n)
    src = fill(layers, planes, 40 * bs, heads, d, dtype=dtype)
    dst = fill(layers, planes, 61 * bs, heads, d, dtype=dtype, seed=1)
    a, b = r.sample(range(40), n), r.sample(range(61), n)
    want = dst.clone()
    for s, t in zip(a, b):
        want[:, :, t * bs:(t + 1) * bs] = src[:, :, s * bs:(s + 1) * bs]
    assert copy_blocks(src, dst, i32(list(zip(a, b))), bs) is dst
    assert same(dst, want)
    # within one pool
    a, b = list(range(20)), r.sample(range(20, 40), 20)
    want = src.clone()
    for s, t in zip(a, b):
        want[:, :, t * bs:(t + 1) * bs] = src[:, :, s * bs:(s + 1) * bs]
    copy_blocks(src, src, i32(list(zip(a, b))), bs)
    assert same(src, want)


def test_copy_between_parts_of_buffers():
    # some layers of a cache, and one plane alone, into pools of their own
    buf, bs = fill(5, 2, 64, 2, 128), 16
    for view in (buf[1:4], buf[:, 1], buf[2, 0], buf[4:5, :1]):
        dst = torch.zeros(*view.shape[:-3], 32, 2, 128, dtype=buf.dtype, device="cuda")
        copy_blocks(view, dst, i32([[3, 0], [1, 1]]), bs)
        assert same(dst[..., :16, :, :], view[..., 48:64, :, :])
        assert same(dst[..., 16:, :, :], view[..., 16:32, :, :])
    with pytest.raises(AssertionError, match="evenly"):
        copy_blocks(buf[:, ::1][:, :1].expand(5, 2, 64, 2, 128), buf, i32([[0, 1]]), bs)


def test_ids_out_of_range_are_skipped():
    src, dst = fill(2, 64, 2, 128), fill(2, 48, 2, 128, seed=1)
    want = dst.clone()
    want[:, 16:32] = src[:, 48:64]
    copy_blocks(src, dst, i32([[-1, 0], [4, 0], [0, 3], [0, -1], [3, 1], [2**31 - 1, 2]]), 16)
    assert same(dst, want)
    copy_blocks(src, dst, torch.empty(0, 2, dtype=torch.int32, device="cuda"), 16)
    assert same(dst, want)


def fork_by_hand(pool, tables, lens, children, bs):
    pool, tables, lens = pool.clone(), tables.clone(), lens.clone()
    old = tables.clone()
    for parent, child, length, new in children:
        w, rest = divmod(length, bs)
        tables[child, :w] = old[parent, :w]
        if rest:
            last = int(old[parent, w])
            tables[child, w] = new
            pool[..., new * bs:new * bs + rest, :, :] = pool[..., last * bs:last * bs + rest, :, :]
        lens[child] = length
    return pool, tables, lens


@pytest.mark.parametrize("layers,planes,heads,d,bs,dtype", SHAPES)
@pytest.mark.parametrize("blocks", [1, 5, 300])
def test_fork(layers, planes, heads, d, bs, dtype, blocks):
    announce(f"fork {layers}x{planes}x{heads}x{d} blocks of {bs} {dtype} {blocks}")
    r = random.Random(blocks)
    pool = fill(layers, planes, (blocks + 12) * bs, heads, d, dtype=dtype)
    ids = r.sample(range(blocks + 12), blocks + 12)
    tables = i32([[-7] * (blocks + 2) for _ in range(20)])
    tables[3, :blocks] = i32(ids[:blocks])
    tables[11, :1] = i32(ids[:1])
    lens = i32([5] * 20)
    # whole and started blocks, one token, the empty history, and a second parent
    full = blocks * bs
    lengths = [full, max(full - 1, 0), full - bs + 1, 0, (blocks // 2) * bs, r.randint(0, full),
               r.randint(0, full)]
    slots = r.sample([s for s in range(20) if s not in (3, 11)], len(lengths) + 1)
    children = [[3, c, n, ids[blocks + i]] for i, (c, n) in enumerate(zip(slots, lengths))]
    children.append([11, slots[-1], min(bs, 7), ids[blocks + 9]])
    want = fork_by_hand(pool, tables, lens, children, bs)
    fork_rows(pool, tables, lens, i32(children), bs)
    for got, expect in zip((pool, tables, lens), want):
        assert same(got, expect)


def test_fork_skips_what_is_out_of_range():
    pool, bs = fill(2, 64, 2, 128), 16
    tables, lens = i32([[0, 1, 9], [-1, -1, -1], [-1, -1, -1]]), i32([33, 0, 0])
    before = pool.clone(), tables.clone(), lens.clone()
    bad = [[0, 3, 5, 2], [-1, 1, 5, 2], [0, 1, -1, 2], [0, 1, 5, 4], [0, 1, 5, -1], [0, 0, 5, 2],
           [0, 1, 49, 2],       # four blocks in tables of three
           [0, 1, 40, 2]]       # the parent's third block is not in the pool
    for child in bad:
        fork_rows(pool, tables, lens, i32([child]), bs)
        for got, expect in zip((pool, tables, lens), before):
            assert same(got, expect), child
    fork_rows(pool, tables, lens, torch.empty(0, 4, dtype=torch.int32, device="cuda"), bs)
    # no started block: the new block is not looked at
    fork_rows(pool, tables, lens, i32([[0, 1, 32, -1]]), bs)
    assert tables.tolist() == [[0, 1, 9], [0, 1, -1], [-1, -1, -1]] and lens.tolist() == [33, 32, 0]
    assert same(pool, before[0])


@pytest.mark.parametrize("layers,planes,heads,d,bs,dtype", SHAPES)
@pytest.mark.parametrize("n,n_rows", [(1, 1), (17, 5), (25, 0), (0, 3)])
def test_move(layers, planes, heads, d, bs, dtype, n, n_rows):
    announce(f"move {layers}x{planes}x{heads}x{d} blocks of {bs} {dtype} {n} {n_rows}")
    r = random.Random(n)
    pool = fill(layers, planes, 60 * bs, heads, d, dtype=dtype)
    src, dst = r.sample(range(30, 60), n), r.sample(range(30), n)
    new_ids = list(range(60))
    for s, t in zip(src, dst):
        new_ids[s] = t
    width = 400
    tables = torch.randint(0, 60, (9, width), dtype=torch.int32, device="cuda")
    slots = r.sample(range(9), n_rows)
    rows = [[s, h] for s, h in zip(slots, (0, width, 1, 257, 30))]
    want, wanted = pool.clone(), tables.clone()
    for s, t in zip(src, dst):
        want[..., t * bs:(t + 1) * bs, :, :] = pool[..., s * bs:(s + 1) * bs, :, :]
    for s, held in rows:
        wanted[s, :held] = i32(new_ids)[tables[s, :held].long()]
    empty = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    move_blocks(pool, tables, i32(rows) if rows else empty,
                i32(list(zip(src, dst))) if n else empty, i32(new_ids), bs)
    assert same(pool, want) and same(tables, wanted)


def test_move_skips_what_is_out_of_range():
    pool = fill(1, 64, 1, 128)
    before = pool.clone()
    tables = i32([[0, 4, -1, 3], [1, 1, 1, 1]])
    move_blocks(pool, tables, i32([[0, 9], [2, 4], [-1, 4]]), i32([[4, 0], [0, 4], [-1, 1]]),
                i32([2, 1, 2, 0]), 16)
    # entries past a row's width are not there, ids that are no blocks stay
    assert tables.tolist() == [[2, 4, -1, 0], [1, 1, 1, 1]] and same(pool, before)


def test_offsets_past_32_bits():
    # planes of 2.2 GB, blocks at their far ends, and more than 2^32 bytes between planes
    bs, heads = 64, 8
    slots = 1100 * 1024 // bs * bs
    buf = torch.zeros(2, 2, slots, heads, 128, dtype=torch.bfloat16, device="cuda")
    last = slots // bs - 1
    buf[..., -bs:, :, :] = fill(2, 2, bs, heads, 128)
    assert buf.stride(0) * 2 > 1 << 32
    copy_blocks(buf, buf, i32([[last, last - 1], [last - 5, 1]]), bs)
    assert same(buf[..., -2 * bs:-bs, :, :], buf[..., -bs:, :, :])
    tables, lens = i32([[last], [0]]), i32([bs, 0])
    fork_rows(buf, tables, lens, i32([[0, 1, bs - 1, last - 2]]), bs)
    assert same(buf[..., -3 * bs:-2 * bs - 1, :, :], buf[..., -bs:-1, :, :])
    assert not buf[..., -2 * bs - 1, :, :].any()
    move_blocks(buf, tables, i32([[0, 1]]), i32([[last, 0]]),
                torch.arange(last + 1, dtype=torch.int32, device="cuda").roll(1), bs)
    assert same(buf[..., :bs, :, :], buf[..., -bs:, :, :]) and tables[0, 0] == last - 1


def test_on_another_stream_and_in_a_graph():
    pool, bs = fill(4, 2, 20 * 16, 2, 128), 16
    tables, lens = i32([[3, 5, 7], [0, 0, 0]]), i32([40, 0])
    children, pairs = i32([[0, 1, 40, 9]]), i32([[1, 11], [2, 12]])
    new_ids, rows = torch.arange(20, dtype=torch.int32, device="cuda"), i32([[0, 3], [1, 3]])

    def step(p, t, ln):
        fork_rows(p, t, ln, children, bs)
        copy_blocks(p, p, pairs, bs)
        move_blocks(p, t, rows, i32_pairs, new_ids, bs)

    i32_pairs = i32([[7, 14]])
    new_ids[7] = 14
    want = [t.clone() for t in (pool, tables, lens)]
    step(*want)
    side = torch.cuda.Stream()
    other = [t.clone() for t in (pool, tables, lens)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*other)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, want):
        assert same(a, b)
    state = [t.clone() for t in (pool, tables, lens)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*state)
    for _ in range(3):
        for a, b in zip(state, (pool, tables, lens)):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(state, want):
            assert same(a, b)
        step(*[t.clone() for t in (pool, tables, lens)])
