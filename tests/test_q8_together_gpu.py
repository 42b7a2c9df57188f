"""8-bit layers at the same time: from two threads, and two captured ones replayed on two streams."""
import threading

import pytest
import torch

import test_q8_gpu as base
from conftest import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"


def layers(m, dtype, count):
    """Layers of 256 x 600 features, one's weights and input each, as calls without arguments."""
    g = torch.Generator().manual_seed(m)
    out = []
    for _ in range(count):
        norm = (1 + 0.1 * torch.randn(256, generator=g)).to(dtype).to(DEV)
        bias = torch.randn(384, generator=g).to(dtype).to(DEV)
        ws = [base.weight_of(g, *size)[2] for size in ((384, 256), (256, 256), (1200, 256, True), (256, 600))]
        x = base.rows_of(g, dtype, m, 256).to(DEV)
        out.append(lambda x=x, norm=norm, ws=ws, bias=bias: base.layer(x, norm, *ws, bias))
    return out


def same(a, b):
    return all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("m", [3, 40, 300])
def test_from_two_threads(m):
    announce(f"8-bit layers from two threads, {m}")
    calls = layers(m, torch.bfloat16, 2)
    want = [f() for f in calls]
    torch.cuda.synchronize()
    failed = []

    def work(f, expected):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = f()
                    torch.cuda.current_stream().synchronize()
                    assert same(got, expected)
        except BaseException as error:
            failed.append(error)
    threads = [threading.Thread(target=work, args=a) for a in zip(calls, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("m", [3, 40, 300])
def test_two_graphs_on_two_streams(m):
    announce(f"8-bit layers in two graphs, {m}")
    calls = layers(m, torch.float16, 2)
    want = [f() for f in calls]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in calls], []
    for graph, f in zip(graphs, calls):
        with torch.cuda.graph(graph):
            outs.append(f())
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                for _ in range(5):
                    graph.replay()
        eager = [f() for f in calls]
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(outs + eager, want + want))
