"""What Qwen2ForCausalLM.quantize_ refuses, on the CPU: no kernel runs here."""
import pytest
import torch
import torch.nn as nn

from model import QwenConfig, Qwen2ForCausalLM

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
