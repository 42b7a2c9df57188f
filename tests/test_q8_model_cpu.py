"""What Qwen2ForCausalLM.quantize_ refuses and what it means to graphs captured before, on the CPU: no kernel runs
here."""
import pickle
from types import SimpleNamespace

import pytest
import torch
import torch.nn as nn

from graphs import DecodeGraphs
from kernels import q8
from kv_cache import KVCache
from model import QwenConfig, Qwen2ForCausalLM, transposed

CFG = QwenConfig(hidden_size=256, num_layers=2, num_heads=2, num_kv_heads=1, intermediate_size=520,
                 vocab_size=512)


@pytest.mark.parametrize("name", ["gate_up_proj", "down_proj"])
def test_a_biased_feed_forward_block_is_refused(name):
    """The block in 8 bits has no bias: quantize_ says so before it replaces anything."""
    model = Qwen2ForCausalLM(CFG).bfloat16()
    mlp = model.layers[1].mlp
    old = getattr(mlp, name)
    setattr(mlp, name, nn.Linear(old.in_features, old.out_features, bias=True).bfloat16())
    with pytest.raises(AssertionError, match="bias"):
        model.quantize_()
    assert not model.quantized
    assert all(type(layer.self_attn.qkv_proj) is nn.Linear for layer in model.layers)


class Graph:
    """A captured graph that counts its replays."""
    replays = 0

    def replay(self):
        self.replays += 1


def graphs_of(model):
    """DecodeGraphs with a one-row graph as captured from model, over a cache that keeps nothing."""
    graphs = object.__new__(DecodeGraphs)
    event = SimpleNamespace(synchronize=lambda: None, record=lambda: None)
    bufs = (torch.zeros(4), torch.zeros(1, 1), torch.zeros(4), torch.zeros(1, 1))
    graph = Graph()
    vars(graphs).update(
        model=model, W=1, buckets=[1], graphs={1: (graph, torch.zeros(1, 1, 5), bufs, event)}, shared_graphs={},
        cache=SimpleNamespace(device_tables=False, SHARED_MAX_ROWS=1, advance=lambda *a: None,
                              pack_step=lambda *a, **k: None))
    graphs._held = graphs._weights()
    return graphs, graph


@pytest.fixture
def stand_in(monkeypatch):
    """quantize_ on the CPU, for what it does around the kernels."""
    monkeypatch.setattr(q8, "quantize_weight", lambda w, gated=False: SimpleNamespace(sig=tuple(w.shape)))


@pytest.mark.parametrize("replace", ["projections", "projections and head", "embeddings"])
def test_graphs_captured_before_weights_are_replaced_do_not_run(replace, stand_in):
    """They read the replaced weights' memory, which is somebody else's by then."""
    model = Qwen2ForCausalLM(CFG).bfloat16()
    graphs, graph = graphs_of(model)
    graphs.run([0], [3])
    with torch.no_grad():
        model.embed_tokens.weight[3] *= 2      # in place: the graph reads it
    graphs.run([0], [3])
    assert graph.replays == 2
    if replace == "embeddings":
        model.embed_tokens.weight = nn.Parameter(model.embed_tokens.weight.detach().clone())
    else:
        model.quantize_(lm_head=replace != "projections")
    with pytest.raises(RuntimeError, match="replaced"):
        graphs.run([0], [3])
    with pytest.raises(RuntimeError, match="replaced"):
        graphs.capture_shared()
    assert graph.replays == 2


def test_graphs_of_a_model_of_another_kind_run():
    graphs, graph = graphs_of(SimpleNamespace(forward_meta=None))
    graphs.run([0], [3])
    assert graph.replays == 1


@pytest.mark.parametrize("lm_head", [False, True])
def test_the_transposed_embeddings_go_with_the_head_that_used_them(lm_head, stand_in):
    model = Qwen2ForCausalLM(CFG).bfloat16()
    transposed(model.embed_tokens.weight)
    model.quantize_(lm_head=lm_head)
    assert hasattr(model.embed_tokens.weight, "_mi_transposed") == (not lm_head)


def test_a_model_saved_before_there_was_quantize_runs():
    """Saved whole, a model comes back with the attributes that it had then."""
    model = Qwen2ForCausalLM(CFG).init_random()
    for name in ("quantized", "head8", "_head8_made", "_replaced"):
        vars(model).pop(name, None)
    old = pickle.loads(pickle.dumps(model))
    caches = [KVCache(8, 16, "cpu", torch.float32, CFG.num_layers, CFG.num_kv_heads, CFG.head_dim) for _ in range(2)]
    ids = torch.arange(5)[None]
    got, want = (m(ids, c, [c.alloc()]) for m, c in zip((old, Qwen2ForCausalLM(CFG).init_random()), caches))
    assert torch.equal(got, want) and old.weights_held()[0] == 0


def test_a_head_that_quantize_did_not_make_is_kept():
    """Set by hand, or saved whole with the model before it was kept what the head was made of."""
    model = Qwen2ForCausalLM(CFG)
    model.head8 = head = SimpleNamespace()
    model.refresh_head8()
    model.refresh_head8()
    assert model.head8 is head
