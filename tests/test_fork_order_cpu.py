"""The order that puts sequences which share blocks side by side (KVCache.order), over forks whose ancestors
come and go: what the cache keeps for it is bounded by the sequences that live."""
import pickle
import random

import pytest
import torch

from kv_cache import KVCache


def cache_of(num_blocks, **kw):
    return KVCache(num_blocks, 16, "cpu", torch.float32, 1, 1, 4, **kw)


def grow(cache, seq, n):
    cache.ensure_capacity(seq, cache.length(seq) + n)
    cache.advance([seq], n)


def books(cache):
    """Bytes of all that the cache keeps on the host beside its buffer."""
    return len(pickle.dumps({k: v for k, v in vars(cache).items() if k != "buf"}))


def test_generations_leave_nothing_behind():
    cache = cache_of(40)
    seq, other = cache.alloc(), cache.alloc()
    grow(cache, seq, 100)
    sizes = []
    for i in range(1500):
        child, = cache.fork(seq)
        cache.free(seq)
        seq = child
        assert cache.order([other, seq]) == [0, 1]
        sizes.append(books(cache))
    assert sizes[-1] <= sizes[20] + 200      # (numbers of more digits)
    # a search that keeps four of eight each time
    beam = [seq] + cache.fork(seq, 3)
    rng = random.Random(1)
    sizes = []
    for i in range(400):
        both = beam + [cache.fork(s)[0] for s in beam]
        assert sorted(cache.order(both)) == list(range(8))
        rng.shuffle(both)
        for s in both[4:]:
            cache.free(s)
        beam = both[:4]
        sizes.append(books(cache))
    assert sizes[-1] <= min(sizes[:50]) + 1000
    for s in beam + [other]:
        cache.free(s)
    empty = cache_of(40)
    assert books(cache) <= books(empty) + 100 and cache._extra == 0


@pytest.mark.parametrize("seed", range(8))
def test_order_keeps_families_together(seed):
    """At every level: what lives of any sequence's family, itself gone or not, stands together, behind
    that sequence; families stand where their first row stood."""
    rng, cache = random.Random(seed), cache_of(4000, max_seqs=400)
    path = {}                       # every sequence that ever was: its ancestors and itself
    live = []
    for _ in range(3):
        s = cache.alloc()
        grow(cache, s, rng.randint(40, 90))
        path[s] = (s,)
        live.append(s)
    for step in range(250):
        s = rng.choice(live)
        if rng.random() < 0.45 and len(live) > 3:
            cache.free(s)
            live.remove(s)
        else:
            for c in cache.fork(s, rng.randint(1, 2)):
                path[c] = path[s] + (c,)
                live.append(c)
                grow(cache, c, rng.randint(1, 20))
        rows = rng.sample(live, rng.randint(1, len(live)))
        order = cache.order(rows)
        assert sorted(order) == list(range(len(rows)))
        got = [rows[i] for i in order]
        if not cache._extra:
            assert got == rows
            continue
        for top in {p for s in rows for p in path[s]}:
            at = [i for i, s in enumerate(got) if top in path[s]]
            assert at == list(range(at[0], at[0] + len(at)))
            assert top not in got or got[at[0]] == top
        roots = [path[s][0] for s in got]
        seen = []
        for s in rows:
            if path[s][0] not in seen:
                seen.append(path[s][0])
        assert list(dict.fromkeys(roots)) == seen
