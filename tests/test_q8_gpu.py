"""Rows, products and feed-forward blocks in 8 bits (csrc/q8_quant.hip, csrc/q8_rows.hip) against their
definition in 64 bits.

Tolerances.  U = 2^-24 is half a step of fp32, relative; H = finfo(t).eps / 2 that of the 16-bit type.
  value   r w, 127 / max|r w| (whose divisor is itself r w rounded) and their product: four roundings of a number
          of at most 127, so a value is within 1/2 + 127 * 4 U of v / scale
  scale   the sum of n squares in fp32: each thread adds at most 64 before the sums join over at most 1024
          threads in 6 + 16 additions: 86 U, halved by the root; mean, eps, root (2 ulp, 4 U) and the
          three operations behind: 60 U for all
  product the whole number rounded to fp32, two factors (each scale exact, or 60 U off), bias and residual:
          8 U of the magnitudes added, then H of the result (or half the least positive number)
"""
import copy

import pytest
import torch

from conftest import announce
from kernels import q8
from kernels.rope import rope_kv_write
from oracle import q8 as o8

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
VALUE, SCALE = 127 * 4 * U, 60 * U
DTYPES = [torch.bfloat16, torch.float16]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the smallest positive number of the type."""
    return torch.finfo(dtype).smallest_normal * half(dtype)


def rows_of(g, dtype, rows, n, spread=1.0):
    x = torch.randn(rows, n, generator=g) * torch.where(torch.rand(n, generator=g) < 0.02, 9.0, 1.0)
    return (x * torch.exp(spread * torch.randn(rows, 1, generator=g))).to(dtype)


def strided(x, pad, at):
    """x on the GPU as a view of rows `pad` elements longer, `at` elements in."""
    buf = torch.full((x.shape[0], x.shape[1] + pad), 3.0, dtype=x.dtype, device=DEV)
    buf[:, at:at + x.shape[1]] = x.to(DEV)
    return buf[:, at:at + x.shape[1]]


def check_rows(got, v, scale_tol=SCALE):
    """got: Rows; v: what they stand for, in 64 bits."""
    ratio, scale = o8.quantize(v)
    values = got.values.cpu()
    R, n = v.shape
    assert got.n == n and values.shape == (R, n) and got.data.numel() == q8.rows_bytes(R, n)
    behind = torch.arange(-(-n // 128) * 128).view(-1, 4, 1, 16) >= n
    live = (torch.arange(-(-R // 16) * 16) < R).view(-1, 1, 1, 16, 1)
    panels = got.data.cpu().view(-1, behind.shape[0], 4, 16, 16)
    assert not (panels.bool() & behind & live).any(), "what lies behind a row is zeros"
    fine = torch.isfinite(scale)
    assert torch.equal(torch.isnan(got.scale.cpu()), ~fine)
    assert not values[~fine].any()
    off = (got.scale.cpu().double() - scale).abs() / scale
    assert (off[fine] <= scale_tol).all(), off[fine].max()
    far = (values[fine, :n].double() - ratio[fine]).abs()
    assert (far <= 0.5 + VALUE).all(), far.max()


SIZES = [(1, 1), (3, 7), (2, 64), (5, 128), (4, 1000), (1, 1536), (130, 1536), (300, 640), (70, 2048), (3, 2049),
         (9, 4864), (2, 8960), (2, 16384), (3, 16385), (1, 40008)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", SIZES)
def test_quantize(rows, n, dtype):
    announce(f"quantize {rows} x {n} {dtype}")
    g = torch.Generator().manual_seed(rows * n)
    x = rows_of(g, dtype, rows, n)
    got = q8.quantize(x.to(DEV))
    check_rows(got, x, 2 * U)
    for pad, at in ((8, 8), (5, 3)):
        again = q8.quantize(strided(x, pad, at))
        assert torch.equal(again.values, got.values) and torch.equal(again.scale, got.scale)
    back = got.dequantize()
    want = got.values.double() * got.scale.double()[:, None]
    assert back.dtype == dtype
    assert ((back.double() - want).abs() <= (half(dtype) + 2 * U) * want.abs() + least(dtype)).all()
    into = strided(torch.zeros(rows, n, dtype=dtype), 3, 1)
    assert torch.equal(got.dequantize(out=into), back)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("add", [False, True])
def test_add_rmsnorm(rows, n, add, dtype):
    announce(f"add_rmsnorm {rows} x {n} add={add} {dtype}")
    g = torch.Generator().manual_seed(rows * n + 1)
    x, y = rows_of(g, dtype, rows, n), rows_of(g, dtype, rows, n)
    w = (1 + 0.2 * torch.randn(n, generator=g)).to(dtype)
    r = o8.add(x, y) if add else x
    xd, yd, wd = x.to(DEV), y.to(DEV) if add else None, w.to(DEV)
    res, got = q8.add_rmsnorm(xd, wd, 1e-6, y=yd)
    assert torch.equal(res.cpu(), r)
    check_rows(got, o8.rmsnorm(r, w, 1e-6))
    assert torch.equal(xd.cpu(), x)
    for xs, ys, out in ((strided(x, 3, 1), strided(y, 5, 2), None),
                        (strided(x, 8, 0), strided(y, 16, 8), "x"),
                        (strided(x, 8, 8), y.to(DEV), "y"), (xd, y.to(DEV), "x")):
        into = {"x": xs, "y": ys, None: None}[out]
        if not add:
            ys, into = None, None
        res, again = q8.add_rmsnorm(xs, wd, 1e-6, y=ys, residual_out=into)
        assert torch.equal(res.cpu(), r)
        assert torch.equal(again.values, got.values)
        # (other loads, other order of the sum)
        assert ((again.scale - got.scale).abs() <= 2 * SCALE * got.scale).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [96, 1003, 5000])
def test_rows_of_nothing_and_of_no_number(n, dtype):
    x = torch.ones(9, n, dtype=dtype)
    x[0] = 0
    x[1] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps    # the least positive number
    x[2, n // 2] = float("inf")
    x[3, -1] = float("nan")
    x[4, 0] = float("-inf")
    x[5] = torch.finfo(dtype).max
    x[6] = 0
    x[6, n - 1] = -2.5
    x[7] *= -1
    got = q8.quantize(x.to(DEV))
    check_rows(got, x, 2 * U)
    assert not got.values[0].any() and (got.values[5] == 127).all()
    assert got.values[6, n - 1] == -127 and (got.values[7] == -127).all()
    w = torch.ones(n, dtype=dtype, device=DEV)
    _, got = q8.add_rmsnorm(x.to(DEV), w, 1e-6)
    bad = torch.isnan(got.scale.cpu())
    # the largest bf16's square is past fp32: its mean is infinite and the row is zero times a number
    assert bad[2:5].all() and not bad[[0, 1, 6, 7, 8]].any()
    assert not got.values[:1].any() and got.scale[0] >= 0
    _, got = q8.add_rmsnorm(x[6:].to(DEV), w, 1e-6)
    check_rows(got, o8.rmsnorm(x[6:], w.cpu(), 1e-6))


@pytest.mark.parametrize("step", [1, 3, 5, 7, 10, 13])
def test_ties_go_to_the_even_number(step):
    # every value is a whole number or one and a half, times the scale: exact in fp16, and so is the answer
    halves = torch.arange(-127, 128).double()
    x = halves * step / 2.0 ** 7
    x[0], x[-1] = -127 * step / 2.0 ** 6, 127 * step / 2.0 ** 6
    assert torch.equal(x.to(torch.float16).double(), x)
    want = torch.round(halves / 2)
    want[0], want[-1] = -127, 127
    x = x.to(torch.float16)[None].to(DEV)
    got = q8.quantize(x)
    assert got.scale.item() == step / 2.0 ** 6
    assert torch.equal(got.values[0].cpu().double(), want)
    # normalised, by a weight of one
    one = torch.ones(255, dtype=torch.float16, device=DEV)
    _, normed = q8.add_rmsnorm(x, one, 1e-6)
    assert torch.equal(normed.values[0].cpu().double(), want)
    # the same in the launch of a product: a weight of ones in one place each gives the values back
    eye = torch.eye(256, dtype=torch.int8)[:, :255].contiguous()
    w = q8.Weight(eye.to(DEV), torch.full((256,), 2.0 ** 6 / step, device=DEV))
    for rows in (x, x.repeat(40, 1)):
        out = q8.linear(rows, w).cpu().double()
        assert torch.equal(out[:, :255], want.expand(len(rows), -1))
        out = q8.linear(rows, w, norm_weight=one, eps=1e-6)
        assert torch.equal(out, q8.linear(q8.add_rmsnorm(rows, one, 1e-6)[1], w))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("n,k", [(2, 1), (16, 64), (34, 100), (130, 130), (1000, 257), (2048, 1536)])
def test_weight_layout(n, k, gated):
    g = torch.Generator().manual_seed(n + k)
    values = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    scale = torch.rand(n, generator=g)
    want = o8.packed(values, gated).flatten()
    for v in (values.to(DEV), strided(values, 5, 3), strided(values, 16, 0)):
        w = q8.Weight(v, scale.to(DEV), gated)
        assert torch.equal(w.data.cpu(), want)
    assert (w.out_features, w.in_features, w.gated) == (n, k, gated)


def weight_of(g, n, k, gated=False):
    values = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    if n * k > 4:
        values.view(-1)[3] = -128
    scale = torch.rand(n, generator=g) * 0.01 / k ** 0.5 + 1e-5
    return values, scale, q8.Weight(values.to(DEV), scale.to(DEV), gated)


def check_product(out, rows, values, scale, bias, residual, extra=0.0):
    """out against the product of Rows; extra: what each entry may be off beside."""
    dt = out.dtype
    q, xs = rows.values.cpu(), rows.scale.cpu()
    want = o8.product(q, xs, values, scale)
    size = want.abs()
    for t in (bias, residual):
        if t is not None:
            want = want + t.double()
            size = size + t.double().abs()
    tol = (8 * U + 2 * SCALE) * size + extra
    tol = tol + half(dt) * (want.abs() + tol) + least(dt)
    got = out.cpu().double()
    over = want.abs() > torch.finfo(dt).max   # (none in these tests)
    assert not over.any()
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


# rows across every tile height, features that end inside panels, in features that end inside steps
PRODUCTS = [(1, 16, 64), (1, 2048, 1536), (2, 1, 1), (3, 17, 129), (15, 48, 96), (16, 1536, 1536), (17, 100, 640),
            (31, 777, 1001), (33, 130, 200), (48, 64, 8960), (64, 2048, 1536), (65, 33, 300),
            (100, 128, 256), (127, 250, 128), (129, 257, 1000), (150, 896, 4864), (200, 1024, 64),
            (257, 513, 520), (300, 1536, 1536), (513, 384, 896), (1025, 300, 1100), (70, 5000, 72),
            (400, 1503, 2100), (50, 8500, 130), (300, 2701, 300), (513, 8300, 72), (1300, 3333, 200),
            (3, 66000, 70), (2, 65553, 2100), (151, 16383, 72), (262, 16323, 600), (644, 16598, 70),
            (517, 13074, 300), (193, 16455, 200), (644, 16405, 300), (771, 16440, 72), (7, 5003, 70),
            (16, 7000, 1300), (5, 17900, 1500), (16, 9001, 1400), (9, 20011, 1900), (12, 20000, 600), (10, 100, 2000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(m, n, k, dtype):
    announce(f"product {m} x {n} x {k} {dtype}")
    g = torch.Generator().manual_seed(m + 3 * n + 7 * k)
    x = rows_of(g, dtype, m, k, 0.3)
    values, scale, w = weight_of(g, n, k)
    bias, res = torch.randn(n, generator=g).to(dtype), torch.randn(m, n, generator=g).to(dtype)
    rows = q8.quantize(x.to(DEV))
    check_product(q8.linear(rows, w), rows, values, scale, None, None)
    check_product(q8.linear(rows, w, bias=bias.to(DEV)), rows, values, scale, bias, None)
    out = q8.linear(rows, w, bias=bias.to(DEV), residual=res.to(DEV))
    check_product(out, rows, values, scale, bias, res)
    # in place, in strided rows whose surroundings stay as they are
    for pad, at in ((8, 8), (7, 3)):
        buf = torch.full((m + 2, n + pad), 3.0, dtype=dtype, device=DEV)
        view = buf[1:m + 1, at:at + n]
        view.copy_(res)
        assert q8.linear(rows, w, bias=bias.to(DEV), residual=view, out=view) is view
        assert torch.equal(view, out)
        view.fill_(3.0)
        assert (buf == 3.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_linear_is_the_product_of_its_rows(m, n, k, dtype):
    announce(f"linear {m} x {n} x {k} {dtype}")
    g = torch.Generator().manual_seed(m + 5 * n + 11 * k)
    x = rows_of(g, dtype, m, k, 0.3)
    values, scale, w = weight_of(g, n, k)
    norm = (1 + 0.2 * torch.randn(k, generator=g)).to(dtype)
    res = torch.randn(m, n, generator=g).to(dtype)
    for xd in (x.to(DEV), strided(x, 8, 8), strided(x, 3, 1)):
        rows = q8.quantize(xd)
        out = q8.linear(xd, w, residual=res.to(DEV))
        check_product(out, rows, values, scale, None, res)
        _, rows = q8.add_rmsnorm(xd, norm.to(DEV), 1e-6)
        out = q8.linear(xd, w, norm_weight=norm.to(DEV), eps=1e-6)
        check_product(out, rows, values, scale, None, None)


def mlp_bounds(rows, gate_up, gate_up_scale, down, down_scale):
    """The block's second product in 64 bits from its first rows, and how far it may be off: whole steps of
    values next to a border, the first product's 8 U + 2 SCALE and what an exponential (8 U) and |g|
    make of it in the activation."""
    q, xs = rows.values.cpu(), rows.scale.cpu()
    both = o8.product(q, xs, gate_up, gate_up_scale)
    gate, up = both.chunk(2, 1)
    act = o8.silu_mul(gate, up)
    ratio, step = o8.quantize(act)
    rel = 8 * U + 2 * SCALE
    off = act.abs() * ((2 + gate.abs()) * rel + 8 * U) / step[:, None]      # in steps
    off = off + ratio.abs() / 127 * off.amax(1, keepdim=True) + VALUE
    near = ((ratio - ratio.floor() - 0.5).abs() <= off).double()
    slack = near @ down.double().abs().t() * step[:, None] * down_scale.double()[None, :]
    amax_rel = (off.amax(1) / 127)[:, None]
    want = o8.product(torch.round(ratio), step, down, down_scale)
    return want, slack + want.abs() * amax_rel


MLPS = [(1, 1536, 8960), (1, 64, 8), (2, 100, 36), (16, 1536, 8960), (5, 128, 17), (17, 896, 4864),
        (33, 300, 500), (64, 256, 1000), (65, 512, 1024), (150, 896, 4864), (260, 640, 1531),
        (515, 256, 768), (130, 512, 1100), (400, 2176, 750), (40, 64, 4201), (600, 128, 3500), (138, 70, 8192),
        (757, 100, 5548), (166, 72, 8203), (2443, 40, 3093), (920, 200, 3081), (1014, 72, 2981), (1239, 40, 6249),
        (2321, 40, 4339), (3, 64, 20000), (40, 48, 33001), (5, 200, 4700), (3, 2000, 3000),
        (15, 1400, 5000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,hidden,inter", MLPS)
def test_mlp(m, hidden, inter, dtype):
    announce(f"mlp {m} x {hidden} x {inter} {dtype}")
    g = torch.Generator().manual_seed(m + 3 * hidden + 7 * inter)
    x = rows_of(g, dtype, m, hidden, 0.3)
    norm = (1 + 0.2 * torch.randn(hidden, generator=g)).to(dtype)
    gu, gus, gate_up = weight_of(g, 2 * inter, hidden, gated=True)
    dn, dns, down = weight_of(g, hidden, inter)
    gus, dns = gus * 3, dns * 3
    gate_up, down = q8.Weight(gu.to(DEV), gus.to(DEV), True), q8.Weight(dn.to(DEV), dns.to(DEV))
    xd, nd = x.to(DEV), norm.to(DEV)

    def check(out, rows, residual):
        want, slack = mlp_bounds(rows, gu, gus, dn, dns)
        size = want.abs()
        if residual is not None:
            want, size = want + residual.double(), size + residual.double().abs()
        tol = (8 * U + 2 * SCALE) * size + slack
        tol = tol + half(dtype) * (want.abs() + tol) + least(dtype)
        far = (out.cpu().double() - want).abs()
        assert (far <= tol).all(), (far / tol).max()

    _, rows = q8.add_rmsnorm(xd, nd, 1e-6)
    out = q8.mlp(xd, gate_up, down, residual=xd, norm_weight=nd, eps=1e-6)
    check(out, rows, x)
    assert torch.equal(xd.cpu(), x)
    check(q8.mlp(xd, gate_up, down), q8.quantize(xd), None)
    for pad, at in ((8, 8), (3, 1)):
        view = strided(x, pad, at)
        assert q8.mlp(view, gate_up, down, residual=view, norm_weight=nd, eps=1e-6, out=view) is view
        # (rows that lie otherwise may have their squares summed in another order: the scale moves in its
        # last places, within SCALE, and activations next to a border by a step, which check() counts)
        check(view, rows, x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,hidden,heads", [(1, 1536, (12, 2)), (16, 1536, (12, 2)), (9, 896, (14, 2)), (5, 1001, (1, 1)),
                                            (16, 2048, (40, 8)), (3, 64, (3, 3)), (17, 256, (4, 1)),
                                            (2, 2049, (2, 1))])
def test_qkv_rope_is_the_separate_launches(m, hidden, heads, dtype):
    announce(f"qkv_rope {m} x {hidden} {heads} {dtype}")
    g = torch.Generator().manual_seed(m + hidden)
    hq, hkv = heads
    _, _, w = weight_of(g, (hq + 2 * hkv) * 128, hidden)
    x = rows_of(g, dtype, m, hidden, 0.3)
    norm = (1 + 0.2 * torch.randn(hidden, generator=g)).to(dtype).to(DEV)
    angle = torch.rand(m, 64, generator=g).repeat(1, 2) * 6.28
    bias = torch.randn(w.out_features, generator=g).to(dtype).to(DEV)
    slots = torch.randperm(40, generator=g)[:m].to(torch.int32)
    if m > 2:
        slots[1], slots[m // 2] = -1, 40      # nowhere
    slots = slots.to(DEV)
    cos16, sin16 = angle.cos().to(dtype), angle.sin().to(dtype)
    one_launch = m <= q8.FUSED_ROWS and hidden <= q8.FUSED_IN
    pad, at = (5, 3) if one_launch else (8, 8)     # (rope_kv_write takes rows at multiples of 16 bytes)
    for xd, cos, sin, b in ((x.to(DEV), cos16.to(DEV), sin16.to(DEV), bias),
                            (strided(x, 3, 1), strided(cos16, pad, at), strided(sin16, pad, at), None)):
        pools = [torch.full((2, 2, 40, hkv, 128), 3.0, dtype=dtype, device=DEV) for _ in range(2)]
        got = q8.qkv_rope(xd, norm, 1e-6, w, b, cos, sin, slots, pools[0][1, 0], pools[0][1, 1], hq, hkv)
        qkv = q8.linear(xd, w, bias=b, norm_weight=norm, eps=1e-6)
        want = rope_kv_write(qkv, cos16.to(DEV), sin16.to(DEV), slots,
                             pools[1][1, 0], pools[1][1, 1], hq, hkv)
        assert torch.equal(got, want) and torch.equal(*pools)


@pytest.mark.parametrize("m", [1, 16, 40, 200])
def test_a_row_that_is_no_number_stays_alone(m):
    g = torch.Generator().manual_seed(m)
    dtype, hidden, inter = torch.bfloat16, 256, 640
    x = rows_of(g, dtype, m, hidden).to(DEV)
    _, _, gate_up = weight_of(g, 2 * inter, hidden, gated=True)
    _, _, down = weight_of(g, hidden, inter)
    norm = torch.ones(hidden, dtype=dtype, device=DEV)
    calls = [lambda t: q8.linear(t, down_t), lambda t: q8.linear(t, down_t, norm_weight=norm, eps=1e-6),
             lambda t: q8.mlp(t, gate_up, down, residual=t, norm_weight=norm, eps=1e-6)]
    _, _, down_t = weight_of(g, inter, hidden)
    clean = [f(x) for f in calls]
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[m // 2, 7] = bad
        for f, want in zip(calls, clean):
            got = f(y)
            assert torch.isnan(got[m // 2]).all()
            keep = [i for i in range(m) if i != m // 2]
            assert torch.equal(got[keep], want[keep])


def test_quantized_weight_is_a_row_for_each_feature():
    g = torch.Generator().manual_seed(3)
    w = torch.randn(50, 200, generator=g).to(torch.bfloat16)
    got = q8.quantize_weight(w.to(DEV))
    rows = q8.quantize(w.to(DEV))
    check_rows(rows, w, 2 * U)
    assert torch.equal(got.data.cpu(), o8.packed(rows.values.cpu()).flatten())
    assert torch.equal(got.scale, rows.scale)


@pytest.mark.parametrize("m,n", [(1, 40), (16, 300), (30, 200), (70, 130), (300, 1000), (600, 2100), (2048, 2100),
                                 (1300, 6200)])
def test_longest_sums(m, n):
    """in_features 131,072 with every value at 127: 2,114,060,288, the largest sum in 32 bits."""
    announce(f"longest sums {m} x {n}")
    g = torch.Generator(device=DEV).manual_seed(m)
    sign_x, sign_w = (torch.randint(0, 2, (c, 1), generator=g, device=DEV) * 2 - 1 for c in (m, n))
    x = (sign_x * 0.375).bfloat16().expand(m, q8.MAX_IN).contiguous()
    scale = torch.rand(n, generator=g, device=DEV) + 0.5
    w = q8.Weight((sign_w * 127).to(torch.int8).expand(n, q8.MAX_IN).contiguous(), scale)
    rows = q8.quantize(x)
    total = (sign_x * sign_w.t() * (127 * 127 * q8.MAX_IN)).float()
    want = (total * rows.scale[:, None] * scale).bfloat16()
    assert torch.equal(q8.linear(rows, w), want) and torch.equal(q8.linear(x, w), want)


def test_most_rows():
    announce("most rows")
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(q8.MAX_ROWS, 24, generator=g, device=DEV, dtype=torch.float16)
    w = q8.quantize_weight(torch.randn(40, 24, generator=g, device=DEV, dtype=torch.float16))
    norm = torch.randn(24, generator=g, device=DEV, dtype=torch.float16)
    assert torch.equal(q8.linear(x, w)[-7:], q8.linear(x[-7:], w))
    r, rows = q8.add_rmsnorm(x, norm, 1e-6, y=x)
    want_r, want = q8.add_rmsnorm(x[-7:].clone(), norm, 1e-6, y=x[-7:])
    assert torch.equal(r[-7:], want_r) and torch.equal(rows.dequantize()[-7:], want.dequantize())
    with pytest.raises(AssertionError):
        q8.quantize(x.new_empty(q8.MAX_ROWS + 1, 1))


def test_past_two_gigabytes():
    """Rows, weights and results that lie more than 2^31 bytes in: the last ones against calls of their own."""
    g = torch.Generator(device=DEV).manual_seed(5)
    n, k, few = 270000, 8192, 37
    announce("rows past 2^31 bytes")
    x = torch.randn(n, k, generator=g, device=DEV, dtype=torch.bfloat16)
    small = q8.quantize_weight(torch.randn(48, k, generator=g, device=DEV, dtype=torch.bfloat16))
    rows, last = q8.quantize(x), q8.quantize(x[-few:].clone())
    assert torch.equal(rows.scale[-few:], last.scale)
    assert torch.equal(rows.dequantize()[-few:], last.dequantize())
    assert torch.equal(q8.linear(rows, small)[-few:], q8.linear(last, small))
    del rows
    announce("weights past 2^31 bytes")
    big, end = q8.quantize_weight(x), q8.quantize_weight(x[-16 * 3:].clone())
    for m in (1, 20, 70, 300):
        y = torch.randn(m, k, generator=g, device=DEV, dtype=torch.bfloat16)
        assert torch.equal(q8.linear(y, big)[:, -48:], q8.linear(y, end))


def test_results_and_activations_past_two_gigabytes():
    g = torch.Generator(device=DEV).manual_seed(6)
    m, few = 300000, 5
    announce("results past 2^31 bytes")
    x = torch.randn(m, 64, generator=g, device=DEV, dtype=torch.bfloat16)
    w = q8.quantize_weight(torch.randn(4096, 64, generator=g, device=DEV, dtype=torch.bfloat16))
    assert torch.equal(q8.linear(x, w)[-few:], q8.linear(x[-few:].clone(), w))
    announce("activations past 2^31 bytes")
    gu = torch.randn(4096, 64, generator=g, device=DEV, dtype=torch.bfloat16)
    down = torch.randn(64, 2048, generator=g, device=DEV, dtype=torch.bfloat16)
    gate_up, down = q8.quantize_weight(gu, gated=True), q8.quantize_weight(down)
    # (as many rows as take the same kernels)
    some = x[-20000:].clone()
    assert torch.equal(q8.mlp(x, gate_up, down)[-few:], q8.mlp(some, gate_up, down)[-few:])


@pytest.mark.parametrize("m", [3, 17, 40, 70])
def test_rows_far_apart(m):
    """x, residual and out with rows 2^30 elements or so apart."""
    g = torch.Generator(device=DEV).manual_seed(m)
    k, n, stride = 256, 300, 2 ** 32 // m + 8
    announce(f"rows far apart {m}")
    buf = torch.empty(m * stride, device=DEV, dtype=torch.bfloat16)

    def far(at, width):
        return torch.as_strided(buf, (m, width), (stride, 1), at)

    x, res = (torch.randn(m, c, generator=g, device=DEV, dtype=torch.bfloat16) for c in (k, n))
    far(0, k).copy_(x)
    far(1000, n).copy_(res)
    norm = torch.randn(k, generator=g, device=DEV, dtype=torch.bfloat16)
    w = q8.quantize_weight(torch.randn(n, k, generator=g, device=DEV, dtype=torch.bfloat16))
    for nw in (None, norm):
        kw = {} if nw is None else dict(norm_weight=nw, eps=1e-6)
        got = q8.linear(far(0, k), w, residual=far(1000, n), out=far(2000, n), **kw)
        assert torch.equal(got, q8.linear(x, w, residual=res, **kw))
    assert torch.equal(far(1000, n), res) and torch.equal(far(0, k), x)
    r, rows = q8.add_rmsnorm(far(0, k), norm, 1e-6, y=far(1000, k), residual_out=far(3000, k))
    want_r, want = q8.add_rmsnorm(x, norm, 1e-6, y=far(1000, k).contiguous())
    assert torch.equal(r, want_r) and torch.equal(rows.scale, want.scale)
    assert torch.equal(rows.values, want.values)


def test_a_weight_copied_and_saved(tmp_path):
    g = torch.Generator().manual_seed(6)
    _, _, w = weight_of(g, 48, 200)
    x = rows_of(g, torch.bfloat16, 3, 200).to(DEV)
    want = q8.linear(x, w)
    other = copy.deepcopy(w)
    assert other.data.data_ptr() != w.data.data_ptr() and other.scale.data_ptr() != w.scale.data_ptr()
    torch.save(w, tmp_path / "w.pt")
    loaded = torch.load(tmp_path / "w.pt", weights_only=False)
    on_cpu = torch.load(tmp_path / "w.pt", weights_only=False, map_location="cpu")
    del w
    assert torch.equal(q8.linear(x, other), want) and torch.equal(q8.linear(x, loaded), want)
    with pytest.raises(AssertionError):
        q8.linear(x, on_cpu)


def test_rows_made_of_their_tensors(tmp_path):
    """Rows put together by hand, copied and saved; tensors that do not belong together are refused."""
    g = torch.Generator().manual_seed(8)
    _, _, w = weight_of(g, 48, 200)
    rows = q8.quantize(rows_of(g, torch.float16, 19, 200).to(DEV))
    want = q8.linear(rows, w)
    torch.save(rows, tmp_path / "rows.pt")
    made = q8.Rows(rows.data.clone(), rows.scale.clone(), 200, torch.float16)
    for other in (made, copy.deepcopy(rows), torch.load(tmp_path / "rows.pt", weights_only=False)):
        assert other.data.data_ptr() != rows.data.data_ptr()
        assert torch.equal(q8.linear(other, w), want) and torch.equal(other.dequantize(), rows.dequantize())
    ok = dict(data=rows.data, scale=rows.scale, n=200, dtype=torch.float16)
    for wrong in (dict(data=rows.data[:-1]), dict(data=rows.data[::2]), dict(data=rows.data.view(torch.uint8)),
                  dict(data=rows.data.cpu()), dict(scale=rows.scale.cpu()), dict(scale=rows.scale[:3]),
                  dict(scale=rows.scale.double()), dict(scale=rows.scale.view(19, 1)), dict(n=0), dict(n=300),
                  dict(dtype=torch.float32)):
        with pytest.raises(AssertionError):
            q8.Rows(**{**ok, **wrong})


def test_a_weight_keeps_its_own_tensors_only():
    w = q8.quantize_weight(torch.randn(64, 640, device=DEV, dtype=torch.bfloat16))
    assert w.data.untyped_storage().nbytes() == 64 * 640 and w.scale.untyped_storage().nbytes() == 64 * 4


def test_no_rows():
    g = torch.Generator().manual_seed(0)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    _, _, w = weight_of(g, 64, 64)
    _, _, gu = weight_of(g, 128, 64, gated=True)
    assert q8.quantize(x).values.shape == (0, 64)
    assert q8.linear(x, w).shape == (0, 64) and q8.linear(q8.quantize(x), w).shape == (0, 64)
    assert q8.mlp(x, gu, w).shape == (0, 64)
    assert q8.add_rmsnorm(x, x.new_ones(64), 1e-6)[1].dequantize().shape == (0, 64)


def layer(x, norm, qkv, o, gate_up, down, bias):
    """One layer's products as the model runs them, attention left out."""
    a = q8.linear(x, qkv, bias=bias, norm_weight=norm, eps=1e-6)
    h = q8.linear(a[:, :o.in_features], o, residual=x)
    h = q8.mlp(h, gate_up, down, residual=h, norm_weight=norm, eps=1e-6)
    r, rows = q8.add_rmsnorm(h, norm, 1e-6, y=x)
    return q8.linear(rows, qkv), r, rows.dequantize()


@pytest.mark.parametrize("m", [1, 7, 16, 50, 180])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_run_of_them_captured_and_replayed(m, dtype):
    """The operators in a row, eager, on another stream and in a graph that is replayed between eager calls with
    new inputs: bitwise the same."""
    announce(f"run of them {m} {dtype}")
    g = torch.Generator().manual_seed(m)
    hidden, inter = 256, 600
    norm = (1 + 0.1 * torch.randn(hidden, generator=g)).to(dtype).to(DEV)
    bias = torch.randn(384, generator=g).to(dtype).to(DEV)
    ws = [weight_of(g, 384, hidden)[2], weight_of(g, hidden, hidden)[2],
          weight_of(g, 2 * inter, hidden, gated=True)[2], weight_of(g, hidden, inter)[2]]
    inputs = [rows_of(g, dtype, m, hidden).to(DEV) for _ in range(4)]
    want = [layer(x, norm, *ws, bias) for x in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [layer(x, norm, *ws, bias) for x in inputs]
    side.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    static = inputs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = layer(static, norm, *ws, bias)
    for again in range(2):
        for x, b in zip(inputs, want):
            static.copy_(x)
            graph.replay()
            eager = layer(inputs[again], norm, *ws, bias)
            torch.cuda.synchronize()
            assert all(torch.equal(s, t) for s, t in zip(outs, b))
            assert all(torch.equal(s, t) for s, t in zip(eager, want[again]))
