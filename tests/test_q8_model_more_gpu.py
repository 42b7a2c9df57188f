"""The model with its projections in 8 bits: biases, the head in every kind of step, weights that change."""
import pytest
import torch
import torch.nn as nn

import test_q8_model_gpu as base
from conftest import announce
from graphs import DecodeGraphs
from kernels import q8
from model import Qwen2ForCausalLM
from test_q8_model_gpu import CFG, cache_for, make, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(3, 1), (2, 20)])
def test_the_output_projections_bias(shape, dtype):
    """A layer's attention with a bias on its output projection and without: the two results are rounded once
    each, so they differ by the bias within half a step of either (and four roundings in fp32 beside)."""
    announce(f"[gpu] biased output projection, {shape} {dtype}")
    model = make(dtype)
    o = model.layers[0].self_attn.o_proj = nn.Linear(256, CFG.hidden_size, bias=True).cuda().to(dtype)
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        o.bias.copy_(torch.randn(CFG.hidden_size, generator=g) * 2)
    model.requires_grad_(False).quantize_()
    attn, norm = model.layers[0].self_attn, model.layers[0].input_layernorm
    B, T = shape
    x = torch.randn(B * T, CFG.hidden_size, generator=g).to(dtype).cuda()
    cos, sin = model.rope_cos_sin(torch.arange(T, device="cuda").expand(B, T), dtype)

    def result():
        cache, res = cache_for(dtype), x.clone()
        meta = cache.prepare([cache.alloc() for _ in range(B)], T, CFG.num_heads)
        attn.q8_step(res, norm, (B, T, CFG.hidden_size), cos, sin, cache, 0, meta)
        return res.cpu().double()
    got, bias = result(), attn.o_proj.bias
    attn.o_proj.bias = None
    without, bias = result(), bias.cpu().double()
    tol = torch.finfo(dtype).eps / 2 * (got.abs() + without.abs()) * 1.01 + 2.0 ** -22 * (got.abs() + bias.abs())
    assert ((got - without - bias).abs() <= tol).all()


def test_the_head_of_a_packed_step():
    """A packed step's logits are the head's product with the norm in front, as an ordinary step's are."""
    announce("[gpu] head in 8 bits of a packed step")
    model = make().quantize_(lm_head=True)
    g = torch.Generator().manual_seed(6)
    x = torch.randn(1, 40, CFG.hidden_size, generator=g).bfloat16().cuda()
    cache = cache_for()
    counts = [1, 1, 30, 8]
    meta = cache.prepare_packed([cache.alloc() for _ in counts], counts)
    model.run_layers = lambda *a: x
    got = model.forward_packed(tokens(g, 40), cache, meta)
    last = x[0, [0, 1, 31, 39]]
    want = q8.linear(last, model.head8, norm_weight=model.norm.weight, eps=CFG.rms_norm_eps)
    assert torch.equal(got, want)


def test_graphs_mixed_steps_and_an_engine_with_the_head(monkeypatch):
    """The runs of a model whose layers alone are in 8 bits, with the head too."""
    quantize_ = Qwen2ForCausalLM.quantize_
    monkeypatch.setattr(Qwen2ForCausalLM, "quantize_", lambda model: quantize_(model, lm_head=True))
    base.test_graphs_and_mixed_steps()
    base.test_an_engine_serves_it()


def test_an_embedding_that_changes_changes_the_head():
    announce("[gpu] head in 8 bits after the embedding changed")
    model = make().quantize_(lm_head=True)
    g = torch.Generator().manual_seed(7)
    ids = tokens(g, 2, 5)

    def logits(m):
        cache = cache_for()
        return m(ids, cache, [cache.alloc(), cache.alloc()])
    def step(graphs, cache):
        return graphs.run([cache.alloc()], [3]).clone()
    cache = cache_for()
    graphs = DecodeGraphs(model, cache, buckets=(1,))
    logits(model)
    step(graphs, cache)
    other = make()
    with torch.no_grad():
        for m in (model, other):
            m.embed_tokens.weight[5:9] *= 3.0
    want = logits(other.quantize_(lm_head=True))
    captured = step(graphs, cache)
    assert torch.equal(logits(model), want)
    c = cache_for()
    assert torch.equal(captured, step(DecodeGraphs(other, c, buckets=(1,)), c))
    # another tensor in its place, of the same values doubled
    for m in (model, other):
        m.embed_tokens.weight = nn.Parameter(m.embed_tokens.weight.detach() * 2, requires_grad=False)
    fresh = make()
    fresh.embed_tokens.weight = nn.Parameter(other.embed_tokens.weight.detach().clone(), requires_grad=False)
    assert torch.equal(logits(model), logits(fresh.quantize_(lm_head=True)))
    # of another size: nothing to bring up to date
    model.embed_tokens.weight = nn.Parameter(torch.cat([model.embed_tokens.weight] * 2), requires_grad=False)
    with pytest.raises(AssertionError, match="as quantize_ saw"):
        logits(model)


def test_a_head_made_in_inference_mode_follows_too():
    model, other = make(), make()
    with torch.inference_mode():
        model.quantize_(lm_head=True)
    ids = tokens(torch.Generator().manual_seed(8), 1, 4)
    with torch.no_grad():
        for m in (model, other):
            m.embed_tokens.weight[5:9] *= 3.0
        got, want = (m(ids, c, [c.alloc()]) for m, c in ((model, cache_for()), (other.quantize_(lm_head=True), cache_for())))
    assert torch.equal(got, want)
