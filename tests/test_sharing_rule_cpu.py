"""Which steps over forked sequences read shared blocks once (KVCache.shared_groups, sharing_pays): measured
steps on both sides of the rule.  The caches are never written, so their memory is never touched."""
import pytest
import torch

from kv_cache import KVCache


def step(heads, groups, own, lone=()):
    """A cache of `heads` kv heads and its rows: groups [(rows, shared tokens)], `own` tokens behind them, then
    rows of their own of lone[i] tokens."""
    blocks = sum(p // 16 + n * (own // 16 + 1) for n, p in groups) + sum(x // 16 + 1 for x in lone)
    cache = KVCache(blocks + 8, 16, "cpu", torch.bfloat16, 1, heads, 128, max_seqs=600)
    seqs = []

    def grow(s, n):
        cache.ensure_capacity(s, cache.length(s) + n)
        cache.advance([s], n)
    for n, p in groups:
        root = cache.alloc()
        grow(root, p)
        family = [root] + (cache.fork(root, n - 1) if n > 1 else [])
        for s in family:
            grow(s, own)
        seqs += family
    for n in lone:
        seqs.append(cache.alloc())
        grow(seqs[-1], n)
    return cache, seqs


@pytest.mark.parametrize("heads,groups,own,lone,want", [
    # faster on the shared kernel (us shared / plain)
    (2, [(64, 31000)], 64, (), True),                 # 37.7 / 250.7
    (2, [(16, 2048)], 64, (), True),                  # 15.5 / 17.0
    (8, [(4, 4096)], 64, (), True),                   # 16.6 / 22.5
    (2, [(64, 2048)], 64, (), True),
    (2, [(8, 16384)], 500, [500] * 56, True),
    # slower there, though 24 MiB and more are saved
    (2, [(64, 512)], 64, (), False),                  # 17.6 / 16.1
    (4, [(64, 256)], 64, (), False),                  # 18.5 / 15.6
    (8, [(32, 256)], 64, (), False),                  # 17.9 / 15.3
    (1, [(256, 256)], 64, (), False),                 # 23.0 / 17.4
    (2, [(4, 16384)], 500, [500] * 252, False),       # 61.5 / 52.4
    (2, [(8, 4096)], 2000, [2000] * 248, False),      # 127.7 / 113.5
    (2, [(2, 4096)], 64, (), False),                  # little saved
])
def test_decode_steps(heads, groups, own, lone, want):
    cache, seqs = step(heads, groups, own, lone)
    assert (cache.shared_groups(seqs) is not None) is want
    cache.SHARED_BYTES = 0
    assert cache.shared_groups(seqs) is not None      # 0: whenever blocks are shared


@pytest.mark.parametrize("heads,rows,prefix,new,splits,want", [
    (2, 8, 8192, 8, True, False),       # 25.9 / 22.5, the keys cut
    (2, 32, 2048, 8, False, True),      # 25.7 / 59.5, not cut
    (2, 4, 31000, 2, True, True),       # 26.0 / 29.8
    (2, 2, 31000, 2, True, False),      # 31.2 / 23.1
    (8, 16, 512, 16, False, False),     # 26.0 / 20.6
    (4, 64, 256, 16, False, False),     # 34.0 / 26.9
    (2, 16, 4096, 4, False, True),
    (4, 16, 8192, 32, True, False),     # 60.3 / 49.6
])
def test_steps_of_several_tokens(heads, rows, prefix, new, splits, want):
    cache, seqs = step(heads, [(rows, prefix // 16 * 16)], 64)
    cache.SHARED_BYTES = 1
    groups = cache.shared_groups(seqs)
    del cache.SHARED_BYTES
    walk = 0 if splits else prefix + 64 + new
    assert cache.sharing_pays(seqs, groups, new * rows, splits, walk) is want


def test_a_short_prompt_beside_many_decoding_rows_earns_nothing():
    """12 MB shared by two of 64 long rows: not worth a decode step, nor with a new conversation's few
    tokens; a message over a long history is worth it."""
    cache, seqs = step(2, [(2, 12288)], 500, [4000] * 62)
    groups = cache._groups(seqs)
    assert not cache.sharing_pays(seqs, groups)
    assert not cache.sharing_pays(seqs, groups, 64 + 19, walk=20)
    assert cache.sharing_pays(seqs, groups, 64 + 19, walk=12288 + 520)
