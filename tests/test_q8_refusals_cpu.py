"""Calls of kernels.q8 that are refused before the GPU is touched, each with a message that says why."""
import pytest
import torch

from kernels import q8


def _rows():
    rows = object.__new__(q8.Rows)
    rows._hold(torch.zeros(q8.rows_bytes(3, 64), dtype=torch.int8), torch.ones(3), 64, torch.bfloat16)
    return rows


def _weight(n, k, gated=False):
    return q8._held(torch.zeros(n * 128, dtype=torch.int8), torch.ones(n), n, k, gated)


@pytest.mark.parametrize("call", [
    lambda x: q8.quantize(x), lambda x: q8.add_rmsnorm(x, torch.ones(64), 1e-6),
    lambda x: q8.mlp(x, _weight(128, 64, True), _weight(64, 64)),
    lambda x: q8.qkv_rope(x, torch.ones(64), 1e-6, _weight(384, 64), None, None, None, None, None, None, 1, 1)])
def test_rows_in_8_bits_go_to_linear_alone(call):
    with pytest.raises(AssertionError, match="rows in 8 bits go to linear"):
        call(_rows())
