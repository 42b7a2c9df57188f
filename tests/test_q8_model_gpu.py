"""The model with its projections in 8 bits (Qwen2ForCausalLM.quantize_): its steps are the operators' in a row, in
every batch shape, captured or not."""
import pytest
import torch

from conftest import announce
from engine import Engine, run_concurrent_chats
from graphs import DecodeGraphs
from kernels import q8
from kernels.fa2 import fa2_paged
from kernels.rope import rope_kv_write
from kv_cache import KVCache
from model import Linear8, QwenConfig, Qwen2ForCausalLM

pytestmark = pytest.mark.gpu
CFG = QwenConfig(hidden_size=256, num_layers=2, num_heads=2, num_kv_heads=1, intermediate_size=520,
                 vocab_size=512)


def make(dtype=torch.bfloat16):
    return (Qwen2ForCausalLM(CFG).cuda().init_random(std=0.05, seed=0).to(dtype).eval()
            .requires_grad_(False))


def cache_for(dtype=torch.bfloat16, blocks=64):
    return KVCache(blocks, 16, "cuda", dtype, CFG.num_layers, CFG.num_kv_heads, CFG.head_dim)


def tokens(g, *shape):
    return torch.randint(0, CFG.vocab_size, shape, generator=g).cuda()


def by_hand(model, ids, cache, seqs):
    """A step as the operators in a row; returns the last positions' logits."""
    (B, T), cfg = ids.shape, model.cfg
    meta = cache.prepare(seqs, T, cfg.num_heads)
    x = model.embed_tokens(ids).view(B * T, -1)
    pos = meta.starts_dev[:, None] + torch.arange(T, device="cuda")[None, :]
    cos, sin = (t[:, 0].reshape(B * T, -1) for t in model.rope_cos_sin(pos, x.dtype))
    for i, layer in enumerate(model.layers):
        attn, mlp = layer.self_attn, layer.mlp
        qkv = q8.linear(x, attn.qkv_proj.weight, bias=attn.qkv_proj.bias,
                        norm_weight=layer.input_layernorm.weight, eps=cfg.rms_norm_eps)
        q = rope_kv_write(qkv, cos, sin, meta.slot_mapping32, cache.k_pool(i), cache.v_pool(i),
                          cfg.num_heads, cfg.num_kv_heads)
        a = fa2_paged(q.view(B, T, cfg.num_heads, -1).transpose(1, 2), cache.k_pool(i), cache.v_pool(i),
                      meta.block_table, meta.kv_lens, block_size=16, max_kv_len=meta.max_kv,
                      is_causal=T > 1).transpose(1, 2).reshape(B * T, -1)
        x = q8.linear(a, attn.o_proj.weight, residual=x)
        x = q8.mlp(x, mlp.gate_up_proj.weight, mlp.down_proj.weight, residual=x,
                   norm_weight=layer.post_attention_layernorm.weight, eps=cfg.rms_norm_eps)
    cache.advance(seqs, T)
    last = x.view(B, T, -1)[:, -1]
    if model.head8 is not None:
        return q8.linear(last, model.head8, norm_weight=model.norm.weight, eps=cfg.rms_norm_eps)
    return None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_step_is_its_operators_in_a_row(dtype):
    announce(f"[gpu] model in 8 bits, {dtype}")
    model = make(dtype).quantize_(lm_head=True)
    mine, hand = cache_for(dtype), cache_for(dtype)
    g = torch.Generator().manual_seed(1)
    rows = 3
    seqs, hseqs = [mine.alloc() for _ in range(rows)], [hand.alloc() for _ in range(rows)]
    for T in (40, 1, 1, 7, 1):
        ids = tokens(g, rows, T)
        got = model(ids, mine, seqs)
        assert torch.equal(got[:, 0], by_hand(model, ids, hand, hseqs))
        assert torch.equal(mine.buf, hand.buf)


def test_near_the_16_bit_model():
    """Rows of n normal numbers reach about 4 of their deviation, so a step is 4 / 127 and its error, uniform, 0.9%
    of them; two such factors 1.3% of a product.  The activation reaches about 15 of its own: 3.4%, and
    3.5% with its weight.  Four products a layer, two layers and the head, as if all met the logits in full: the
    root of 2 (3 * 1.3^2 + 3.5^2) + 1.3^2, 6.1%."""
    ref, model = make(), make().quantize_(lm_head=True)
    g = torch.Generator().manual_seed(2)
    ca, cb = cache_for(), cache_for()
    a, b = [ca.alloc() for _ in range(4)], [cb.alloc() for _ in range(4)]
    for T in (50, 1):
        ids = tokens(g, 4, T)
        want, got = ref(ids, ca, a).float(), model(ids, cb, b).float()
        assert torch.isfinite(got).all()
        assert ((got - want).norm() / want.norm()).item() < 0.1


def test_graphs_and_mixed_steps():
    announce("[gpu] model in 8 bits: graphs, mixed steps")
    model = make().quantize_()
    g = torch.Generator().manual_seed(3)

    def near(got, want):
        # attention's parts meet in another order: a value next to a border may step, 1/127 of its row's
        # largest, which two layers carry on
        assert torch.isfinite(got).all()
        assert (got.float() - want.float()).abs().max().item() < 0.05 * want.float().abs().max().item()
    plain, captured, mixed = cache_for(), cache_for(), cache_for()
    sets = [[c.alloc() for _ in range(5)] for c in (plain, captured, mixed)]
    prompts = tokens(g, 5, 30)
    for cache, seqs in zip((plain, captured, mixed), sets):
        model(prompts, cache, seqs)
    graphs = DecodeGraphs(model, captured, buckets=(8,))
    for step in range(4):
        ids = tokens(g, 5, 1)
        want = model(ids, plain, sets[0])[:, 0]
        near(graphs.run(sets[1], ids[:, 0].tolist()), want)
        new = mixed.alloc()
        got = model.forward_mixed([[t] for t in ids[:, 0].tolist()] + [prompts[0].tolist()], mixed,
                                  sets[2] + [new])
        near(got[:5], want)
        mixed.free(new)


def test_an_engine_serves_it():
    announce("[gpu] engine over a model in 8 bits")
    model = make().quantize_()
    cache = cache_for(blocks=128)
    engine = Engine(model, cache, max_reply_tokens=8, seed=0,
                    decode_graphs=DecodeGraphs(model, cache, buckets=(1, 2, 4)))
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, CFG.vocab_size, (n,), generator=g).tolist() for n in (40, 7, 300, 96)]
    assert run_concurrent_chats(engine, prompts, reply_tokens=8)["tokens"] == 32
    assert cache.free_block_count() == 128


def test_refusals():
    model = make().quantize_()
    with pytest.raises(AssertionError):
        model.quantize_()
    assert type(model.layers[0].mlp.down_proj) is Linear8
    other = make()
    other.layers[1].mlp.down_proj.register_forward_hook(lambda *a: None)
    with pytest.raises(AssertionError):
        other.quantize_()
    assert not other.quantized
    assert all(type(layer.mlp.gate_up_proj) is torch.nn.Linear for layer in other.layers)
    hooked = make().quantize_()
    hooked.layers[0].mlp.down_proj.register_forward_hook(lambda *a: None)
    cache = cache_for()
    with pytest.raises(AssertionError):
        hooked(torch.zeros(1, 3, dtype=torch.long, device="cuda"), cache, [cache.alloc()])


def test_hooked_attention_runs_module_by_module():
    """With something hooked on, the modules are called one by one: the norm's output is rounded on the way to 8
    bits, which changes values next to a border by a step."""
    model, hooked = make().quantize_(), make().quantize_()
    calls = []
    hooked.layers[0].self_attn.o_proj.register_forward_hook(lambda *a: calls.append(1))
    g = torch.Generator().manual_seed(4)
    ids = tokens(g, 2, 9)
    ca, cb = cache_for(), cache_for()
    want = model(ids, ca, [ca.alloc(), ca.alloc()]).float()
    got = hooked(ids, cb, [cb.alloc(), cb.alloc()]).float()
    assert calls == [1]
    # (6.1% is what all of the values' steps come to, see above)
    assert ((got - want).norm() / want.norm()).item() < 0.061
