"""Forked sequences on the CPU: KVCache.fork / copy_from / compact against a plain record of what
every sequence holds, the counts of holders behind free blocks, the groups of rows that share, and
Engine.fork against a recomputation of each branch's history."""
import random

import pytest
import torch

from engine import Conversation, Engine
from kv_cache import KVCache
from test_engine_cpu import tiny_cache, tiny_model


def small_cache(num_blocks=40, **kw):
    return KVCache(num_blocks, 16, "cpu", torch.float32, 2, 1, 4, **kw)


def append(cache, seq, n, g):
    """Append n tokens of random K and V; returns them as [layers, 2, n, 1, 4]."""
    meta = cache.prepare([seq], n)
    new = torch.randn(2, 2, n, 1, 4, generator=g)
    for layer in range(2):
        cache.write(layer, meta, *(new[layer, i].transpose(0, 1)[None] for i in (0, 1)))
    cache.advance([seq], n)
    return new


def held(cache, seq):
    n = cache.length(seq)
    return torch.stack([torch.stack(cache.read_row(layer, cache._block_tables[seq], n)).transpose(1, 2)
                        for layer in range(2)])


def check(cache, want):
    counts = [0] * cache.num_blocks
    for s, w in want.items():
        assert torch.equal(held(cache, s), w), s
        for b in cache._block_tables[s]:
            counts[b] += 1
    assert counts == cache._holders
    assert cache._extra == sum(c - 1 for c in counts if c)
    assert sorted(cache._free_blocks) == [b for b, c in enumerate(counts) if c == 0]


@pytest.mark.parametrize("seed", range(6))
def test_random_forks_trims_frees_and_compactions_keep_every_history(seed):
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    cache, other = small_cache(max_seqs=24), small_cache(60)
    want = {}
    for _ in range(160):
        op = rng.choice(["new", "append", "append", "fork", "fork", "free", "trim", "compact", "copy"])
        some = rng.choice(list(want)) if want else None
        try:
            if op == "new":
                want[cache.alloc()] = torch.zeros(2, 2, 0, 1, 4)
            elif some is None:
                continue
            elif op == "append":
                n = rng.randint(1, 40)
                need = cache.blocks_needed(some, cache.length(some) + n)
                if need <= cache.free_block_count():
                    want[some] = torch.cat([want[some], append(cache, some, n, g)], dim=2)
            elif op == "fork":
                n, length = rng.randint(1, 3), rng.choice([None, rng.randint(0, cache.length(some))])
                for s in cache.fork(some, n, length):
                    want[s] = want[some][:, :, :length]
            elif op == "free":
                cache.free(some)
                del want[some]
            elif op == "trim":
                if cache.free_block_count() > 2:
                    cache.ensure_capacity(some, cache.length(some) + 20)
                cache.trim(some)
            elif op == "compact":
                n = cache.compact()
                assert n == cache.num_blocks - cache.free_block_count()
                assert all(b < n for t in cache._block_tables.values() for b in t)
            else:
                there = other.copy_from(cache, some)
                assert torch.equal(held(other, there), want[some])
                other.free(there)
        except RuntimeError:     # no blocks or no slots left: nothing changed
            pass
        check(cache, want)
    for s in list(want):
        cache.free(s)
    assert cache.free_block_count() == cache.num_blocks and cache._extra == 0


def test_branches_write_into_blocks_of_their_own():
    cache, g = small_cache(), torch.Generator().manual_seed(1)
    a = cache.alloc()
    first = append(cache, a, 37, g)
    b, c = cache.fork(a, 2)
    assert cache._block_tables[b][:2] == cache._block_tables[c][:2] == cache._block_tables[a][:2]
    assert len({t[2] for t in map(cache._block_tables.get, (a, b, c))}) == 3
    tails = [append(cache, s, 3, g) for s in (b, a, c)]
    for s, tail in zip((b, a, c), tails):
        assert torch.equal(held(cache, s), torch.cat([first, tail], dim=2))
    # a history that ends with a block needs no copy
    d = cache.fork(a, 1, 32)[0]
    assert cache._block_tables[d] == cache._block_tables[a][:2] and cache.length(d) == 32
    e = cache.fork(a, 1, 0)[0]
    assert cache._block_tables[e] == [] and cache.length(e) == 0


def test_refused_forks_change_nothing():
    cache, g = small_cache(5, max_seqs=3), torch.Generator().manual_seed(1)
    a = cache.alloc()
    append(cache, a, 40, g)
    before = (list(cache._free_blocks), list(cache._holders), list(cache._free_slots))
    for n, length, error in ((3, None, RuntimeError), (3, 32, RuntimeError), (0, None, ValueError),
                             (-1, None, ValueError), (1, 41, ValueError), (1, -1, ValueError),
                             (1.5, None, TypeError), (1, 16.0, TypeError)):
        with pytest.raises(error):
            cache.fork(a, n, length)
        assert before == (cache._free_blocks, cache._holders, cache._free_slots)
    with pytest.raises(KeyError):
        cache.fork(7)
    with pytest.raises(RuntimeError):
        small_cache(2).copy_from(cache, a)
    for bad in (KVCache(9, 32, "cpu", torch.float32, 2, 1, 4), KVCache(9, 16, "cpu", torch.float16, 2, 1, 4),
                KVCache(9, 16, "cpu", torch.float32, 3, 1, 4), KVCache(9, 16, "cpu", torch.float32, 2, 2, 4)):
        with pytest.raises(ValueError):
            bad.copy_from(cache, a)


def test_copy_from_its_own_cache_shares_nothing():
    cache, g = small_cache(), torch.Generator().manual_seed(1)
    a = cache.alloc()
    first = append(cache, a, 37, g)
    b = cache.copy_from(cache, a)
    assert torch.equal(held(cache, b), first) and cache._extra == 0
    assert not set(cache._block_tables[a]) & set(cache._block_tables[b])


def test_reclaimable_counts_blocks_that_no_other_sequence_holds():
    cache, g = small_cache(), torch.Generator().manual_seed(1)
    a = cache.alloc()
    append(cache, a, 40, g)
    b, c = cache.fork(a, 2)
    assert cache.reclaimable([a]) == 1 and cache.reclaimable([a, b]) == 2
    assert cache.reclaimable([a, b, c]) == 5 and cache.reclaimable([]) == 0


def test_groups_cover_what_neighbouring_rows_share():
    cache, g = small_cache(200), torch.Generator().manual_seed(1)
    cache.SHARED_BYTES = 0
    a, lone = cache.alloc(), cache.alloc()
    append(cache, lone, 20, g)
    append(cache, a, 100, g)
    assert cache.shared_groups([a, lone]) is None and cache.order([a, lone]) == [0, 1]
    b, c = cache.fork(a, 2)
    append(cache, b, 30, g)
    d, = cache.fork(b)
    seqs = [d, lone, a, c, b]
    seqs = [seqs[i] for i in cache.order(seqs)]
    # in the order of the tree of forks, where its first row was
    assert seqs == [a, b, d, c, lone]
    cu, prefix = cache.shared_groups(seqs)
    assert (cu, prefix) == ([0, 4, 5], [96, 0])
    # a pair that shares more than the rest is worth its own group only while it saves more
    assert cache.shared_groups([b, d]) == ([0, 2], [128])
    assert cache.shared_groups([lone, b, d]) == ([0, 1, 3], [0, 128])
    assert cache.shared_groups([a]) is None
    del cache.SHARED_BYTES
    assert cache.shared_groups(seqs) is None     # too little to save


@pytest.mark.parametrize("seed", range(4))
def test_groups_of_random_trees_hold_the_same_blocks(seed):
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    cache = small_cache(600)
    cache.SHARED_BYTES = 0
    seqs = [cache.alloc() for _ in range(3)]
    for _ in range(30):
        s = rng.choice(seqs)
        append(cache, s, rng.randint(1, 50), g)
        seqs += cache.fork(s, 1, rng.choice([None, rng.randint(0, cache.length(s))]))
    rng.shuffle(seqs)
    order = cache.order(seqs)
    assert sorted(order) == list(range(len(seqs)))
    rows = [cache._block_tables[seqs[i]] for i in order]
    cu, prefix = cache.shared_groups([seqs[i] for i in order])
    assert cu[0] == 0 and cu[-1] == len(rows) and len(prefix) == len(cu) - 1
    for x, y, p in zip(cu, cu[1:], prefix):
        assert x < y and p % 16 == 0 and len({tuple(t[:p // 16]) for t in rows[x:y]}) == 1
        assert all(len(t) >= p // 16 for t in rows[x:y])
        assert y - x > 1 or p == 0


# -- the engine -----------------------------------------------------------------------------------
def _engine(num_blocks, mixed, model=None):
    # cold enough that the likeliest token is drawn
    return Engine(model or tiny_model(), tiny_cache(num_blocks=num_blocks), max_reply_tokens=6,
                  temperature=1e-6, mixed_prefill=mixed)


@pytest.mark.parametrize("mixed", [False, True])
def test_branches_reply_as_if_they_had_their_own_history(mixed):
    eng = _engine(64, mixed)
    conv = Conversation()
    eng.submit(conv, list(range(50)))
    eng.run_until_idle()
    branches = eng.fork(conv, 3)
    new = [[7, 8], [9], list(range(20))]
    jobs = [eng.submit(c, ids) for c, ids in zip(branches, new)] + [eng.submit(conv, [1, 2])]
    history = list(conv.ids)
    eng.run_until_idle()
    for job, ids in zip(jobs, new + [[1, 2]]):
        alone = _engine(64, mixed, eng.model)
        plain = alone.submit(Conversation(ids=list(history)), ids)
        alone.run_until_idle()
        assert job.generated == plain.generated and len(job.generated) == 6
    for c in branches + [conv]:
        eng.release(c)
    assert eng.cache.free_block_count() == 64


@pytest.mark.parametrize("mixed", [False, True])
def test_a_branch_of_a_running_reply_needs_no_message(mixed):
    eng = _engine(64, mixed)
    conv = Conversation()
    job = eng.submit(conv, list(range(30)))
    for _ in range(3):
        eng.tick()
    at = len(conv.ids)
    branch, = eng.fork(conv)
    again = eng.submit(branch, [])
    eng.run_until_idle()
    # the same history, the likeliest token each time: the same continuation
    rest = job.generated[at - 30:]
    assert rest and again.generated[:len(rest)] == rest
    assert branch.seq is not None and conv.seq is not None


def test_forks_without_room_start_without_cache():
    eng = _engine(6, False)
    conv, idle = Conversation(), Conversation()
    eng.submit(idle, list(range(10)), 2)
    eng.run_until_idle()
    eng.submit(conv, list(range(50)), 2)
    eng.run_until_idle()
    assert idle.seq is not None and eng.cache.free_block_count() == 1
    # two started blocks: the idle conversation makes room for the second
    forks = eng.fork(conv, 2)
    assert idle.seq is None and all(c.seq is not None for c in forks)
    # three more can't be had, also without the first two
    forks = eng.fork(forks[0], 6)
    assert all(c.seq is None for c in forks)
    assert eng.fork(conv, 0) == []
    job = eng.submit(forks[0], [1], 2)
    eng.run_until_idle()
    assert len(job.generated) == 2


def test_idle_branches_make_room():
    """Branches of the conversation that needs room hold blocks it keeps: evicting them gives back what
    is theirs alone, and that is enough."""
    eng = _engine(10, False)
    conv = Conversation()
    eng.submit(conv, list(range(66)), 3)
    eng.run_until_idle()
    branches = eng.fork(conv, 3)
    assert eng.cache.free_block_count() == 2
    assert eng.cache.reclaimable([c.seq for c in branches]) == 3
    job = eng.submit(conv, [5] * 60, 6)      # 70 + 60 + 6 + 1 tokens: 9 blocks, 5 held
    assert eng._fits_after_eviction(job)
    eng.run_until_idle()
    assert len(job.generated) == 6
    # the least recently used went, and no more than had to
    assert [c.seq is None for c in branches] == [True, True, False]
