"""Forks of any size (CPU: the launches are recorded).  A call is cut into launches that the library
takes."""
import torch

from kernels import blocks
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
