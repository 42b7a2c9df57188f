"""Rows and products in 8 bits from their definition, in 64 bits on the CPU."""
import torch

LEAST = 2.0 ** -100   # a row's largest magnitude counts as at least this


def add(x, y):
    """The residual stream as it is stored: the sum rounded to the tensors' type."""
    return (x.double() + y.double()).to(x.dtype)


def rmsnorm(x, weight, eps):
    x = x.double()
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight.double()


def quantize(v):
    """(v / scale before it is rounded, scale [rows]); a row that is not finite has scale NaN."""
    v = v.double()
    scale = v.abs().amax(-1).clamp_min(LEAST) / 127
    scale = torch.where(torch.isfinite(v).all(-1), scale, torch.full_like(scale, float("nan")))
    return v / scale[:, None], scale


def product(values, scale, w, w_scale):
    """values [rows, in], w [out, in] whole numbers, scale [rows], w_scale [out] -> [rows, out]."""
    whole = values.to(torch.float64) @ w.to(torch.float64).t()   # below 2^53: exact
    return whole * scale.double()[:, None] * w_scale.double()[None, :]


def silu_mul(gate, up):
    return gate / (1 + torch.exp(-gate)) * up


def packed(values, gated=False):
    """A weight's values [out, in] as the kernels read them, [panels, steps of 64, 4, 16 rows, 16]."""
    n, k = values.shape
    kp = -(-k // 128) * 128
    if gated:
        half = n // 2
        panels = -(-half // 8)
        full = torch.zeros(2, panels * 8, kp, dtype=torch.int8)
        full[0, :half, :k], full[1, :half, :k] = values[:half], values[half:]
        rows = full.view(2, panels, 8, kp).transpose(0, 1).reshape(panels, 16, kp)
    else:
        panels = -(-n // 16)
        full = torch.zeros(panels * 16, kp, dtype=torch.int8)
        full[:n, :k] = values
        rows = full.view(panels, 16, kp)
    return rows.view(panels, 16, kp // 64, 4, 16).permute(0, 2, 3, 1, 4).contiguous()
