"""A decoder layer's products in 8 bits, sized for timing: the RMSNorm that leaves its rows in 8 bits,
the product of such rows with 8-bit weights, and the gated feed-forward block made of both.

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare` makes what
a program holds before the call, `run` is one pass (in plain torch operations, or with `own` set
through the framework's entry points), `work` says what a pass cannot do without and `exact` gives
the same outputs in 64 bits.

Rows of activations have one scale each, the largest magnitude over 127, taken anew in every call;
weights have one for each output feature and are in 8 bits before the call, as a quantised
checkpoint holds them.  The shapes are Qwen2.5-1.5B's layers (1536 -> 2048 and 2 x 8960, vocabulary
151,936), those of smaller and larger layers, and odd ones.
"""
import math
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # one chat's token between two projections: nothing but latency
        {"name": "norm_1", "kind": "norm", "rows": 1, "hidden": 1536, "add": True, "dtype": "bf16"},
        # a mixed step's rows, of a width that is no multiple of anything
        {"name": "norm_701x1003_fp16", "kind": "norm", "rows": 701, "hidden": 1003, "add": False,
         "dtype": "fp16"},
        # many prompts packed into one step
        {"name": "norm_16384", "kind": "norm", "rows": 16384, "hidden": 1536, "add": True,
         "dtype": "bf16"},
        # one chat's q/k/v projection behind its norm
        {"name": "linear_1", "kind": "linear", "rows": 1, "in": 1536, "out": 2048, "norm": True,
         "bias": True, "residual": False, "dtype": "bf16"},
        # the next tokens' logits of 16 chats, the largest weight there is
        {"name": "linear_16_head", "kind": "linear", "rows": 16, "in": 1536, "out": 151936,
         "norm": True, "bias": False, "residual": False, "dtype": "bf16"},
        # a short prompt, odd in every size
        {"name": "linear_37_odd_fp16", "kind": "linear", "rows": 37, "in": 1001, "out": 777,
         "norm": False, "bias": True, "residual": True, "dtype": "fp16"},
        # the q/k/v projection of a long prompt
        {"name": "linear_4096", "kind": "linear", "rows": 4096, "in": 1536, "out": 2048,
         "norm": True, "bias": True, "residual": False, "dtype": "bf16"},
        # the output projection of a larger layer over a batch of prompts
        {"name": "linear_6001_wide", "kind": "linear", "rows": 6001, "in": 4096, "out": 6144,
         "norm": False, "bias": False, "residual": True, "dtype": "bf16"},
        # one chat's feed-forward block
        {"name": "mlp_1", "kind": "mlp", "rows": 1, "hidden": 1536, "inter": 8960, "dtype": "bf16"},
        # a decode step of 16 chats
        {"name": "mlp_16", "kind": "mlp", "rows": 16, "hidden": 1536, "inter": 8960,
         "dtype": "bf16"},
        # a chat's next message in a smaller layer
        {"name": "mlp_150_fp16", "kind": "mlp", "rows": 150, "hidden": 896, "inter": 4864,
         "dtype": "fp16"},
        # a long prompt's
        {"name": "mlp_4001", "kind": "mlp", "rows": 4001, "hidden": 1536, "inter": 8960,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _size(rng, lo, hi):
    """A width: mostly whole multiples of 128 or 32, as layers have them, one in four odd."""
    n = _log(rng, lo, hi)
    unit = rng.choice([1, 32, 128, 128])
    return max(lo, n // unit * unit)


def draw(rng):
    kind = rng.choice(["norm", "linear", "linear", "mlp", "mlp"])
    most = [work(c) for c in listed() if c["kind"] == kind]
    while True:
        case = _drawn(rng, kind)
        need = work(case)
        if all(need[k] <= max(w[k] for w in most) for k in need):
            return case


def _drawn(rng, kind):
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "norm":
        return {"kind": kind, "rows": _log(rng, 1, 16384), "hidden": _size(rng, 64, 8192),
                "add": rng.random() < 0.5, "dtype": dtype}
    if kind == "linear":
        return {"kind": kind, "rows": _log(rng, 1, 8192), "in": _size(rng, 64, 8960),
                "out": _size(rng, 64, 151936 if rng.random() < 0.1 else 17920),
                "norm": rng.random() < 0.5, "bias": rng.random() < 0.5,
                "residual": rng.random() < 0.5, "dtype": dtype}
    return {"kind": kind, "rows": _log(rng, 1, 8192), "hidden": _size(rng, 64, 4096),
            "inter": _size(rng, 64, 14336), "dtype": dtype}


# -- inputs ---------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _activations(g, dtype, rows, n):
    """Rows of a residual stream: a hundredth of the features several times as large as the rest,
    the rows of different sizes."""
    feature = torch.where(torch.rand(n, generator=g, device=DEV) < 0.01, 6.0, 1.0)
    row = torch.exp(0.5 * _randn(g, rows, 1))
    return (_randn(g, rows, n) * feature * row).to(dtype)


def _weight(g, out, n):
    """A quantised weight as a checkpoint holds it: int8 [out, in] and a scale for each row."""
    w = _randn(g, out, n) * 0.02
    scale = w.abs().amax(1) / 127
    return torch.round(w / scale[:, None]).to(torch.int8), scale


def _norm(g, dtype, n):
    return (1 + 0.1 * _randn(g, n)).to(dtype)


def prepare(case, seed):
    kind, g, dtype = case["kind"], _gen(seed), DTYPES[case["dtype"]]
    s = {"kind": kind}
    rows, n = case["rows"], case["in"] if kind == "linear" else case["hidden"]
    s["x"] = _activations(g, dtype, rows, n)
    if kind == "norm":
        s["norm"] = _norm(g, dtype, n)
        s["y"] = _activations(g, dtype, rows, n) if case["add"] else None
        return s
    if kind == "linear":
        out = case["out"]
        s["norm"] = _norm(g, dtype, n) if case["norm"] else None
        s["bias"] = _randn(g, out).to(dtype) if case["bias"] else None
        s["residual"] = _activations(g, dtype, rows, out) if case["residual"] else None
        weights = {"w": _weight(g, out, n)}
    else:
        s["norm"] = _norm(g, dtype, n)
        weights = {"gate_up": _weight(g, 2 * case["inter"], n), "down": _weight(g, n, case["inter"])}
    if own:
        q8 = _framework()   # laid out once, as a program does when it loads its model
        weights = {k: q8.Weight(*w, gated=k == "gate_up") for k, w in weights.items()}
    s.update(weights)
    return s


def _framework():
    if "my-inference-engine_amd" not in sys.path:
        sys.path.insert(0, "my-inference-engine_amd")
    from kernels import q8
    return q8


# -- one pass -------------------------------------------------------------------------------------
def run(state):
    s, kind = state, state["kind"]
    if own:
        q8 = _framework()
        if kind == "norm":
            r, rows = q8.add_rmsnorm(s["x"], s["norm"], EPS, y=s["y"])
            return r, rows.dequantize(), rows.scale
        if kind == "linear":
            return q8.linear(s["x"], s["w"], bias=s["bias"], residual=s["residual"],
                             norm_weight=s["norm"], eps=EPS)
        return q8.mlp(s["x"], s["gate_up"], s["down"], residual=s["x"], norm_weight=s["norm"],
                      eps=EPS)
    x, dtype = s["x"], s["x"].dtype
    if kind == "norm":
        # the residual stream is kept in the tensors' type, and what is kept is normalised
        r = x if s["y"] is None else (x.float() + s["y"].float()).to(dtype)
        q, scale = _quantized(_normed(r.float(), s["norm"]))
        return r, (q * scale).to(dtype), scale[:, 0]
    h = x.float() if s["norm"] is None else _normed(x.float(), s["norm"])
    if kind == "linear":
        out = _product(h, s["w"])
        if s["bias"] is not None:
            out = out + s["bias"].float()
        if s["residual"] is not None:
            out = out + s["residual"].float()
        return out.to(dtype)
    gate, up = _product(h, s["gate_up"]).chunk(2, 1)
    return (_product(gate / (1 + torch.exp(-gate)) * up, s["down"]) + x.float()).to(dtype)


def _normed(x, weight):
    return x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * weight.float()


def _quantized(x):
    """Rows x in 8 bits: whole numbers of at most 127 (in x's type) and a scale for each row."""
    scale = x.abs().amax(1, keepdim=True) / 127
    return torch.round(x / scale), scale


def _product(x, weight):
    values, scale = weight
    q, row_scale = _quantized(x)
    return torch.matmul(q, values.float().t().contiguous()) * row_scale * scale


# -- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    rows = case["rows"]
    if case["kind"] == "norm":
        n = case["hidden"]
        # x (and y, and their sum written), the norm's weight; the 8-bit rows and their scales
        return {"bytes": rows * n * (7 if case["add"] else 3) + 2 * n + 4 * rows,
                "flops": 6 * rows * n}
    if case["kind"] == "linear":
        n, out = case["in"], case["out"]
        return {"bytes": n * out + 4 * out + 2 * rows * (n + out) + 2 * n * case["norm"]
                + 2 * out * case["bias"] + 2 * rows * out * case["residual"],
                "flops": 2 * rows * n * out}
    n, inter = case["hidden"], case["inter"]
    return {"bytes": 3 * n * inter + 8 * inter + 4 * n + 2 * n + 4 * rows * n,
            "flops": 6 * rows * n * inter}


# -- the same in 64 bits --------------------------------------------------------------------------
def _norm64(x, weight):
    x = x.double()
    return x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * weight.double()


def _linear64(x, values, scale):
    x = x.double()
    step = x.abs().max(-1, keepdim=True).values / 127
    return (x / step).round() @ values.double().t().contiguous() * (step * scale.double())


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    x, dtype = s["x"], s["x"].dtype
    if case["kind"] == "norm":
        total = x.double() if s["y"] is None else x.double() + s["y"].double()
        n = _norm64(total.to(dtype), s["norm"])
        step = n.abs().max(-1, keepdim=True).values / 127
        return total, (n / step).round() * step, step.squeeze(-1)
    h = x.double() if s["norm"] is None else _norm64(x, s["norm"])
    if case["kind"] == "linear":
        out = _linear64(h, *s["w"])
        for t in (s["bias"], s["residual"]):
            if t is not None:
                out = out + t.double()
        return out
    both = _linear64(h, *s["gate_up"])
    inter = case["inter"]
    act = torch.nn.functional.silu(both[:, :inter]) * both[:, inter:]
    return x.double() + _linear64(act, *s["down"])
