"""Captured decode steps over branches (graphs.DecodeGraphs): their sharing graphs are captured beforehand
where that is asked for, and a step for whose graph there is no memory runs on the ordinary one."""
import pytest
import torch

from conftest import announce
from graphs import DecodeGraphs
from kv_cache import KVCache
from test_engine_gpu import SMALL, make
from test_fork_gpu import close

pytestmark = pytest.mark.gpu


def start(n=3):
    model, _ = make("cuda", torch.bfloat16)
    cache = KVCache(100, 16, "cuda", torch.bfloat16, SMALL.num_layers, SMALL.num_kv_heads,
                    SMALL.head_dim, max_blocks_per_seq=16)
    cache.SHARED_BYTES = 0
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(0, SMALL.vocab_size, (1, 100), generator=g).cuda()
    root = cache.alloc()
    with torch.no_grad():
        model(prompt, cache, [root])
    return model, cache, [root] + cache.fork(root, n - 1), g


def steps(model, cache, seqs, graphs, g):
    """Three decode steps, each against the same one of copies that share nothing."""
    for _ in range(3):
        alone = [cache.copy_from(cache, s) for s in seqs]
        t = torch.randint(0, SMALL.vocab_size, (len(seqs), 1), generator=g)
        with torch.no_grad():
            want = torch.cat([model(t[i:i + 1].cuda(), cache, [s])[:, -1] for i, s in enumerate(alone)])
        for s in alone:
            cache.free(s)
        close(graphs.run(seqs, t.flatten().tolist()), want)


def test_captured_beforehand(monkeypatch):
    announce("[gpu] sharing graphs captured beforehand")
    model, cache, seqs, g = start()
    graphs = DecodeGraphs(model, cache, buckets=(2, 4))
    assert not graphs.shared_graphs
    graphs.capture_shared(3)
    assert set(graphs.shared_graphs) == {4}
    graphs.capture_shared()
    assert set(graphs.shared_graphs) == {2, 4}
    monkeypatch.setattr(graphs, "_capture", None)      # no step captures
    steps(model, cache, seqs, graphs, g)
    steps(model, cache, seqs[:2], graphs, g)
    graphs.capture_shared()


@pytest.mark.parametrize("hidden", [False, True])
def test_without_memory_a_step_runs_on_the_ordinary_graph(monkeypatch, hidden):
    announce("[gpu] a sharing graph that cannot be had")
    model, cache, seqs, g = start()
    graphs = DecodeGraphs(model, cache, buckets=(4,))
    asked = []

    def refuse(rows, shared=False):
        asked.append(rows)
        try:
            raise torch.OutOfMemoryError("no memory")
        finally:
            if hidden:                  # as the end of a capture may
                raise RuntimeError("capture ended")
    capture = graphs._capture
    monkeypatch.setattr(graphs, "_capture", refuse)
    steps(model, cache, seqs, graphs, g)
    assert asked == [4] and not graphs.shared_graphs     # not tried at every step
    with pytest.raises(RuntimeError):
        graphs.capture_shared()
    monkeypatch.setattr(graphs, "_capture", capture)     # there is memory again
    graphs.capture_shared()
    assert set(graphs.shared_graphs) == {4}
    steps(model, cache, seqs, graphs, g)


def test_other_errors_are_raised(monkeypatch):
    model, cache, seqs, _ = start()
    graphs = DecodeGraphs(model, cache, buckets=(4,))
    lengths = [cache.length(s) for s in seqs]

    def fail(rows, shared=False):
        raise RuntimeError("something else")
    monkeypatch.setattr(graphs, "_capture", fail)
    with pytest.raises(RuntimeError, match="something else"):
        graphs.run(seqs, [1, 2, 3])
    assert lengths == [cache.length(s) for s in seqs]


def test_a_capture_that_fails_is_waited_for(monkeypatch):
    """A warm-up step that runs out of memory leaves the one before it running on the capture stream, over
    buffers that are free then: what follows on this stream waits for it."""
    model, cache, seqs, g = start()
    graphs = DecodeGraphs(model, cache, buckets=(4,))
    waits, run, calls = [], model.forward_meta, []

    wait = torch.cuda.Stream.wait_stream

    def noted(self, other):
        waits.append(other)
        wait(self, other)
    monkeypatch.setattr(torch.cuda.Stream, "wait_stream", noted)

    def second_fails(*args):
        calls.append(args)
        if len(calls) == 2:
            raise torch.OutOfMemoryError("no memory")
        return run(*args)
    monkeypatch.setattr(model, "forward_meta", second_fails)
    with pytest.raises(torch.OutOfMemoryError):
        graphs.capture_shared()
    assert len(calls) == 2 and waits[-1] == graphs._side
    monkeypatch.undo()
    steps(model, cache, seqs, graphs, g)


def test_host_tables_capture_none():
    model, _ = make("cuda", torch.bfloat16)
    cache = KVCache(100, 16, "cuda", torch.bfloat16, SMALL.num_layers, SMALL.num_kv_heads,
                    SMALL.head_dim, max_blocks_per_seq=16, device_tables=False)
    graphs = DecodeGraphs(model, cache, buckets=(2,))
    graphs.capture_shared()
    assert not graphs.shared_graphs
