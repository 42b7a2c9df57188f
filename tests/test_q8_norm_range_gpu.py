"""Rows at the ends of the norm's range: squares past fp32 or below it, magnitudes below the least that counts."""
import pytest
import torch

import test_q8_gpu as base
from conftest import announce
from kernels import q8
from kernels.model_ops import add_rmsnorm

pytestmark = pytest.mark.gpu
DEV, U = "cuda", 2.0 ** -24


def products(x, w, norm, eps):
    """What is normalised on its way to a product, in a launch of its own and with it."""
    _, rows = q8.add_rmsnorm(x, norm, eps)
    return rows, [q8.linear(rows, w), q8.linear(x, w, norm_weight=norm, eps=eps)]


@pytest.mark.parametrize("m", [1, 3, 16, 40, 200])
@pytest.mark.parametrize("n", [200, 2104])
def test_squares_past_fp32(m, n):
    """A finite row whose mean is infinite: zeros, as of the 16-bit norm; the rows beside it as without it."""
    announce(f"norm past fp32 {m} x {n}")
    g = torch.Generator().manual_seed(m)
    x = base.rows_of(g, torch.bfloat16, m, n).to(DEV)
    norm = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    _, _, w = base.weight_of(g, 48, n)
    _, clean = products(x, w, norm, 1e-6)
    at = m // 2
    x[at] = torch.where(torch.arange(n, device=DEV) % 2 == 0, 3e20, -1e30)
    assert torch.isfinite(x).all() and not add_rmsnorm(x, norm, 1e-6)[1][at].any()
    rows, outs = products(x, w, norm, 1e-6)
    assert rows.scale[at] == 0 and not rows.dequantize()[at].any()
    keep = [i for i in range(m) if i != at]
    for out, want in zip(outs, clean):
        assert not out[at].any() and torch.equal(out[keep], want[keep])


@pytest.mark.parametrize("m", [1, 16, 40])
def test_mean_and_eps_of_nothing(m):
    """A row of zeros without eps is no number, as of the 16-bit norm; the rows beside it are."""
    g = torch.Generator().manual_seed(m)
    x = base.rows_of(g, torch.float16, m, 96).to(DEV)
    x[0] = 0
    norm = torch.ones(96, dtype=torch.float16, device=DEV)
    _, _, w = base.weight_of(g, 48, 96)
    assert torch.isnan(add_rmsnorm(x, norm, 0.0)[1][0]).all()
    rows, outs = products(x, w, norm, 0.0)
    assert torch.isnan(rows.dequantize()[0]).all()
    for out in outs:
        assert torch.isnan(out[0]).all() and torch.isfinite(out[1:]).all()


def test_magnitudes_below_the_least():
    """The largest |r w| counts as at least 2^-100: the scale is that times rsqrt(mean + eps) / 127 (the squares are
    below fp32, so the mean is 0) within the root's 4 U and three operations, the values whole multiples of it."""
    r = torch.full((1, 64), 2.0 ** -103, dtype=torch.bfloat16)
    r[0, 1] = -2.0 ** -101
    r[0, 2] = 0
    _, rows = q8.add_rmsnorm(r.to(DEV), torch.ones(64, dtype=torch.bfloat16, device=DEV), 1e-6)
    eps = torch.tensor(1e-6).double()
    want = 2.0 ** -100 * eps.rsqrt() / 127
    assert abs(rows.scale.item() - want.item()) <= 7 * U * want.item()
    assert rows.values[0, :4].tolist() == [16, -64, 0, 16]      # 127 / 8 = 15.9, 127 / 2 = 63.5 to the even number
