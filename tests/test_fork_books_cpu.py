"""Forks, copies and compactions of any size, and ones whose launch fails (CPU: the launches are recorded or
made to fail).  A call is cut into launches that the library takes; a cache whose copy failed holds what it
held."""
import pytest
import torch

from kernels import blocks
from test_fork_cpu import append, check, held, small_cache
from test_split_workspace import on_gpu


def test_a_fork_of_many_children_goes_out_in_several_launches(monkeypatch):
    calls = []
    monkeypatch.setattr(blocks, "call", lambda device, fn, *args: calls.append(args))
    bs, planes, n = 128, 160, 4096                   # 256 KB a block and plane: 16 pieces of 16 KB
    pool = on_gpu(80, 2, 2 * bs, 8, 128)
    tables, lens = (torch.zeros(*s, dtype=torch.int32) for s in ((n + 1, 4), (n + 1,)))
    children = torch.zeros(n, 4, dtype=torch.int32)
    blocks.fork_rows(pool, tables, lens, children, bs)
    seen = 0
    for args in calls:
        at, count = args[-2:]
        assert at == children.data_ptr() + 16 * seen and count > 0
        # mi_cache_fork_rows takes it: below 2^23 work-groups
        assert count * 16 < (1 << 23) // planes - count // planes - 1
        seen += count
    assert seen == n and len(calls) == 2
    for m in (1, 7):
        calls.clear()
        blocks.fork_rows(pool, tables, lens, children[:m], bs)
        assert [args[-1] for args in calls] == [m]
    calls.clear()
    blocks.fork_rows(pool, tables, lens, children[:0], bs)
    assert not calls


class Full(Exception):
    pass


def fail(*args, **kw):
    raise Full


@pytest.mark.parametrize("length", [37, 32])
def test_a_fork_that_fails_leaves_the_books(monkeypatch, length):
    cache, g = small_cache(), torch.Generator().manual_seed(1)
    a = cache.alloc()
    want = {a: append(cache, a, 37, g)}
    b, = cache.fork(a)
    want[b] = want[a]
    slots = sorted(cache._free_slots)
    cache.device_tables = True               # as on the GPU, up to the upload
    cache.dev_tables = cache.dev_lens = None
    monkeypatch.setattr(cache, "_upload", fail)
    with pytest.raises(Full):
        cache.fork(a, 3, length)
    check(cache, want)
    assert sorted(cache._free_slots) == slots and cache.order([b, a]) == [1, 0]
    cache.device_tables = False
    monkeypatch.setattr(cache, "_copy", fail)
    with pytest.raises(Full):
        cache.fork(a, 3, 37)
    check(cache, want)
    assert sorted(cache._free_slots) == slots


def test_a_copy_that_fails_leaves_the_books(monkeypatch):
    cache, other, g = small_cache(), small_cache(), torch.Generator().manual_seed(1)
    a = cache.alloc()
    want = append(cache, a, 37, g)
    slots = sorted(other._free_slots)
    monkeypatch.setattr(other, "_copy", fail)
    with pytest.raises(Full):
        other.copy_from(cache, a)
    check(other, {})
    assert sorted(other._free_slots) == slots
    assert torch.equal(held(cache, a), want)


@pytest.mark.parametrize("on_device", [False, True])
def test_a_compaction_that_fails_leaves_the_books(monkeypatch, on_device):
    cache, g = small_cache(), torch.Generator().manual_seed(1)
    seqs = [cache.alloc() for _ in range(4)]
    want = {s: append(cache, s, 40, g) for s in seqs}
    for s in seqs[::2]:
        cache.free(s)
        del want[s]
    cache.device_tables, cache.dev_tables = on_device, None
    monkeypatch.setattr(cache, "_upload" if on_device else "_copy", fail)
    with pytest.raises(Full):
        cache.compact()
    check(cache, want)
    monkeypatch.undo()
    cache.device_tables = False
    assert cache.compact() == 6
    check(cache, want)
