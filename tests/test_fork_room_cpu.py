"""Whose cache makes room for forks and for messages beside them (Engine on the CPU): nobody's if it could
not be enough, and not that of branches whose blocks others go on holding."""
import pytest
import torch

from engine import Conversation, Engine
from kv_cache import KVCache
from test_engine_cpu import TINY, tiny_model


def engine(num_blocks, **kw):
    cache = KVCache(num_blocks, 16, "cpu", torch.float32, TINY.num_layers, TINY.num_kv_heads,
                    TINY.head_dim, **kw)
    return Engine(tiny_model(), cache, max_reply_tokens=2, temperature=1e-6, sep_ids=(1,))


def idle(eng, n):
    """An idle conversation with n tokens in the cache, the last of its history beside them."""
    conv = Conversation(ids=list(range(n + 1)))
    conv.seq = eng.cache.alloc()
    eng.cache.ensure_capacity(conv.seq, n)
    eng.cache.advance([conv.seq], n)
    eng._touch(conv)
    return conv


def state(eng):
    return list(eng.resident), eng.cache.free_block_count(), eng.cache.free_slot_count()


def test_a_refused_fork_evicts_nobody():
    eng = engine(20)
    convs = [idle(eng, 30) for _ in range(5)]     # two blocks each: 10 are free, 8 the others'
    before = state(eng)
    for n in (19, 200):                           # a started block for each
        assert all(c.seq is None for c in eng.fork(convs[0], n))
        assert state(eng) == before and all(c.seq is not None for c in convs)
    # as many as can be had, and no more evicted than that takes
    assert all(c.seq is not None for c in eng.fork(convs[0], 11))
    assert [c.seq is None for c in convs] == [False, True, False, False, False]
    eng = engine(20)
    convs = [idle(eng, 30) for _ in range(5)]
    assert all(c.seq is not None for c in eng.fork(convs[0], 18))
    assert eng.cache.free_block_count() == 0


def test_a_fork_refused_for_slots_evicts_nobody():
    eng = engine(60, max_seqs=4)
    convs = [idle(eng, 30) for _ in range(3)]
    before = state(eng)
    assert all(c.seq is None for c in eng.fork(convs[2], 4))
    assert state(eng) == before
    forks = eng.fork(convs[2], 3)       # one slot free, two conversations in the way
    assert all(c.seq is not None for c in forks) and convs[0].seq is None and convs[1].seq is None


@pytest.mark.parametrize("by_fork", [False, True])
def test_branches_that_would_give_back_nothing_stay(by_fork):
    eng = engine(9)
    conv = idle(eng, 48)
    branches = eng.fork(conv, 2)        # whole blocks, all of them the conversation's too
    eng._touch(conv)
    lone, other = idle(eng, 30), idle(eng, 40)    # 1 block is left
    assert [c.seq is None for c in branches] == [False, False] and eng.cache.free_block_count() == 1
    if by_fork:
        assert all(c.seq is not None for c in eng.fork(other, 2))
    else:
        job = eng.submit(Conversation(), list(range(40)), 2)    # 3 blocks
        eng.run_until_idle()
        assert len(job.generated) == 2
    assert lone.seq is None and all(c.seq is not None for c in (conv, other, *branches))


def test_branches_go_where_only_all_of_them_help():
    """Branches that share blocks with each other alone: none gives back anything by itself."""
    eng = engine(7)
    conv = idle(eng, 48)
    branches = eng.fork(conv, 2)
    eng.release(conv)
    assert [eng.cache.reclaimable([c.seq]) for c in branches] == [0, 0]
    job = eng.submit(Conversation(), list(range(80)), 2)    # 6 of 7 blocks
    eng.run_until_idle()
    assert len(job.generated) == 2 and all(c.seq is None for c in branches)


def test_conversations_are_told_apart_without_comparing_histories():
    """Branches have long equal histories: finding one among the others looks at none of them."""
    class Ids(list):
        def __eq__(self, other):
            raise AssertionError("histories compared")
        __hash__ = None

    eng = engine(20)
    conv = idle(eng, 48)
    convs = eng.fork(conv, 3) + [conv]
    for c in convs:
        c.ids = Ids(c.ids)
    eng._touch(convs[1])
    assert [id(c) for c in eng.resident] == [id(convs[i]) for i in (3, 0, 2, 1)]
    more = eng.fork(convs[2], 2)
    eng.release(convs[0])
    assert [id(c) for c in eng.resident] == [id(c) for c in (convs[3], convs[2], convs[1], *more)]
    eng.active = [eng.submit(c, [7], 2) for c in (convs[2], convs[1])]
    last = eng.active[1]
    eng._finish(last)
    assert len(eng.active) == 1 and eng.active[0].conv is convs[2] and eng.finished[-1] is last
