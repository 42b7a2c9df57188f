"""Forked sequences on the GPU: the device tables and pools after fork, copy_from and compact
against a host-table cache on the CPU that sees the same operations (equality: integers and copies),
and the model over branches (fork, decode, chunks, compact, copy to another cache), eager and in
graphs, whose attention reads the shared blocks once, against the same steps reading them for each row.

Two roundings of the same steps differ by what bf16 leaves (a unit in the last place per rounded
value, 2^-8 relative, through two layers): the bar of the graph tests, 2 % of the largest logit."""
import random

import pytest
import torch

from conftest import announce
from engine import Conversation, Engine
from graphs import DecodeGraphs
from kv_cache import KVCache
from test_engine_gpu import SMALL, make

pytestmark = pytest.mark.gpu


def pools_equal(host, dev):
    torch.cuda.synchronize()
    got = dev.buf.cpu()
    for s, table in host._block_tables.items():
        assert dev._block_tables[s] == table
        n = host.length(s)
        idx = torch.tensor([table[p // 16] * 16 + p % 16 for p in range(n)], dtype=torch.long)
        assert torch.equal(got[:, :, idx], host.buf[:, :, idx]), s
        if dev.device_tables:
            slot = dev.slot[s]
            assert dev.dev_tables[slot, :len(table)].tolist() == table
            assert dev.dev_lens[slot].item() == n


@pytest.mark.parametrize("tables", [False, True])
@pytest.mark.parametrize("seed", range(3))
def test_pools_and_tables_follow_the_host_cache(tables, seed):
    announce(f"[gpu] random forks, tables {tables} seed {seed}")
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)

    def mk(n, device, dt):
        return KVCache(n, 16, device, torch.bfloat16, 2, 2, 128, device_tables=dt, max_seqs=16)
    host, dev, there = mk(48, "cpu", False), mk(48, "cuda", tables), mk(64, "cuda", tables)
    host_there = mk(64, "cpu", False)
    host.buf.copy_(torch.randn(host.buf.shape, generator=g))
    dev.buf.copy_(host.buf)
    seqs = []
    for step in range(60):
        op = rng.choice(["new", "append", "append", "fork", "fork", "free", "trim", "compact", "copy"])
        some = rng.choice(seqs) if seqs else None
        try:
            if op == "new":
                a, b = host.alloc(), dev.alloc()
                assert a == b
                seqs.append(a)
            elif some is None:
                continue
            elif op == "append":
                n = rng.randint(1, 40)
                if host.blocks_needed(some, host.length(some) + n) > host.free_block_count():
                    continue
                new = torch.randn(2, 2, 1, 2, n, 128, generator=g).to(torch.bfloat16)
                for c in (host, dev):
                    meta = c.prepare([some], n)
                    for layer in range(2):
                        c.write(layer, meta, *new[layer].to(c.device))
                    c.advance([some], n)
            elif op == "fork":
                n, length = rng.randint(1, 3), rng.choice([None, rng.randint(0, host.length(some))])
                made = host.fork(some, n, length)
                assert made == dev.fork(some, n, length)
                seqs += made
            elif op == "free":
                host.free(some)
                dev.free(some)
                seqs.remove(some)
            elif op == "trim":
                host.trim(some)
                dev.trim(some)
            elif op == "compact":
                assert host.compact() == dev.compact()
            else:
                a, b = host_there.copy_from(host, some), there.copy_from(dev, some)
                assert a == b
                pools_equal(host_there, there)
                host_there.free(a)
                there.free(b)
        except RuntimeError:
            continue
        if step % 5 == 4:
            pools_equal(host, dev)
    pools_equal(host, dev)


def close(got, want):
    got, want = got.float(), want.float()
    assert torch.isfinite(got).all()
    assert (got - want).abs().max().item() <= 0.02 * want.abs().max().item()


def watch(cache):
    """What cache's steps are given to share, as they are prepared."""
    met, inner = [], cache._shared_rows

    def spy(*args):
        met.append(inner(*args))
        return met[-1]
    cache._shared_rows = spy
    return met


def branches(model, cache, prompt, n, tails, share):
    """`prompt` prefilled once (share) and forked, or once per branch; then each branch's tail."""
    seqs = [cache.alloc()]
    model(prompt, cache, seqs)
    if share:
        seqs += cache.fork(seqs[0], n - 1)
    else:
        for _ in range(n - 1):
            seqs.append(cache.alloc())
            model(prompt, cache, seqs[-1:])
    for s, t in zip(seqs, tails):
        if t.numel():
            model(t, cache, [s])
    return seqs


@pytest.mark.parametrize("tables", [False, True])
def test_branches_together_as_they_are_used(tables):
    """Fork, tails, decode steps, a chunk for every row, a mixed step, compact, a copy to another
    cache, decode there: each step's logits equal those of rows that share nothing."""
    g = torch.Generator().manual_seed(5)
    model, _ = make("cuda", torch.bfloat16)

    def mk(n):
        return KVCache(n, 16, "cuda", torch.bfloat16, SMALL.num_layers, SMALL.num_kv_heads,
                       SMALL.head_dim, device_tables=tables)

    def ids(*shape):
        return torch.randint(0, SMALL.vocab_size, shape, generator=g)
    prompt = ids(1, 203).cuda()
    tails = [ids(1, n).cuda() for n in (0, 3, 40, 17, 1)]
    plain, shared, target = mk(160), mk(80), mk(80)
    shared.SHARED_BYTES = target.SHARED_BYTES = 0
    announce(f"[gpu] branches of one history, device tables {tables}")
    with torch.no_grad():
        ps = branches(model, plain, prompt, 5, tails, False)
        ss = branches(model, shared, prompt, 5, tails, True)
        met = watch(shared)

        def both(T):
            t = ids(5, T).cuda()
            close(model(t, shared, ss), model(t, plain, ps))
            assert met[-1].rows == 5 and plain._extra == 0
        for _ in range(3):
            both(1)
        both(7)
        both(1)
        # a mixed step: leading rows with few new tokens (those share), a prompt behind them
        extra = [c.alloc() for c in (plain, shared)]
        rows = [ids(n).tolist() for n in (1, 1, 5, 1, 2, 90)]
        close(model.forward_mixed(rows, shared, ss + extra[1:]),
              model.forward_mixed(rows, plain, ps + extra[:1]))
        assert met[-1].rows == 5 and met[-1].max_q == 5
        # holes, closed again
        for c, s in zip((plain, shared), extra):
            c.free(s)
        plain.free(ps.pop(1))
        shared.free(ss.pop(1))
        ps.append(plain.alloc())
        model(prompt, plain, ps[-1:])
        ss += shared.fork(ss[0], 1, 203)
        used = shared.compact()
        assert used == 80 - shared.free_block_count()
        both(1)
        # one branch and its fork go on in another cache
        moved = target.copy_from(shared, ss[2])
        ms = [moved] + target.fork(moved)
        t = ids(2, 1).cuda()
        want = model(t[:1].expand(2, 1).contiguous(), plain, [ps[2], ps[3]])[:1]
        got = model(t[:1].expand(2, 1).contiguous(), target, ms)
        close(got, want.expand_as(got))
    torch.cuda.synchronize()


def test_graphs_of_sharing_steps_match_eager_ones():
    """Captured decode steps over branches (padded buckets, groups that come and go between replays,
    eager work and forks in between) against eager steps that read every row's blocks."""
    g = torch.Generator().manual_seed(6)
    model, _ = make("cuda", torch.bfloat16)

    def mk(n):
        return KVCache(n, 16, "cuda", torch.bfloat16, SMALL.num_layers, SMALL.num_kv_heads,
                       SMALL.head_dim, max_blocks_per_seq=32)
    plain, shared = mk(200), mk(100)
    shared.SHARED_BYTES = 0
    announce("[gpu] decode graphs over branches")
    graphs = DecodeGraphs(model, shared, buckets=(2, 4, 8))
    prompt = torch.randint(0, SMALL.vocab_size, (1, 150), generator=g).cuda()
    tails = [torch.randint(0, SMALL.vocab_size, (1, n), generator=g).cuda() for n in (0, 5, 30)]
    with torch.no_grad():
        ps = branches(model, plain, prompt, 3, tails, False)
        ss = branches(model, shared, prompt, 3, tails, True)

        def step(rows):
            t = torch.randint(0, SMALL.vocab_size, (len(rows), 1), generator=g)
            want = model(t.cuda(), plain, [ps[i] for i in rows])[:, -1]
            close(graphs.run([ss[i] for i in rows], t.flatten().tolist()), want)
        for _ in range(4):
            step([0, 1, 2])
        assert set(graphs.shared_graphs) == {4}
        step([0])
        step([2, 1])
        # a conversation of its own beside them, then more branches of one of them
        for c, s in ((plain, ps), (shared, ss)):
            s.append(c.alloc())
            model(prompt[:, :33], c, s[-1:])
        for _ in range(2):
            step([0, 1, 2, 3])
            step([3, 0])
        n = plain.length(ps[1])
        ss += shared.fork(ss[1], 2)
        for _ in range(2):
            ps.append(plain.copy_from(plain, ps[1]))
        assert plain.length(ps[-1]) == shared.length(ss[-1]) == n
        for _ in range(3):
            step([0, 2, 1, 4, 5, 3])
        shared.compact()
        for _ in range(3):
            step([0, 2, 1, 4, 5, 3])
        # the others gone, the rest shares nothing
        for i in (0, 1, 4, 5):
            shared.free(ss[i])
        assert shared._extra == 0
        step([2, 3])
    assert set(graphs.shared_graphs) == {2, 4, 8}


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("captured", [False, True])
def test_engine_branches_share_and_complete(mixed, captured):
    """Branches of one conversation through the engine, cold enough to draw the likeliest token,
    complete with the blocks they share read once, and every block comes back."""
    announce(f"[gpu] engine branches: mixed {mixed} captured {captured}")
    model, cache = make("cuda", torch.bfloat16, num_blocks=128)
    cache.SHARED_BYTES = 0
    eng = Engine(model, cache, max_reply_tokens=6, mixed_prefill=mixed,
                 decode_graphs=DecodeGraphs(model, cache, buckets=(1, 4)) if captured else None)
    conv = Conversation()
    eng.submit(conv, list(range(100)))
    eng.run_until_idle()
    forks = eng.fork(conv, 3)
    jobs = [eng.submit(c, new) for c, new in zip(forks + [conv], ([], [5], list(range(30)), [7, 8]))]
    seen = []
    inner = cache.shared_groups

    def spy(seqs):
        seen.append(inner(seqs))
        return seen[-1]
    cache.shared_groups = spy
    eng.run_until_idle()
    assert any(s is not None and len(s[0]) == 2 and s[0][-1] > 1 for s in seen)
    assert all(len(j.generated) == 6 for j in jobs)
    for c in forks + [conv]:
        eng.release(c)
    assert cache.free_block_count() == 128
