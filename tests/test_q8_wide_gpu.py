"""The 8-bit kernels at sizes of wide layers (in features past 2,048), at long rows and at every variant of the few-row
kernel, against the same 64-bit forms and bounds as in test_q8_gpu.py.

A norm's scale there allows 86 additions in the sum of squares, 64 of them a thread's.  Rows past 16,384 (and past 32,768
where there are few) are taken by 1,024 threads, n / 1024 squares each: 128 at the longest row of 131,072, so 150
additions, 75 U of the root and the 17 U behind it: 92 U.
"""
import pytest
import torch

import test_q8_gpu as base
from conftest import announce
from kernels import q8
from oracle import q8 as o8

pytestmark = pytest.mark.gpu
DEV = "cuda"
LONGEST = 92 * base.U

SIZES = [(70, 2100), (130, 4096), (66, 5000), (70, 7001), (65, 8960), (67, 11111), (66, 13000), (200, 16384), (130, 16500),
         (2, 30000)]
PRODUCTS = [(1, 4100, 2200), (16, 6144, 4096), (7, 5003, 9000), (31, 4000, 2300), (20, 900, 2500), (20, 555, 1301),
            (29, 1111, 1900), (47, 3001, 2001)]
MLPS = [(9, 1300, 700), (14, 1900, 900), (5, 1000, 3000), (1, 2100, 1000), (1, 4096, 3000), (3, 2500, 1900),
        (4, 2300, 9500), (1, 2200, 12288), (16, 3584, 1200), (16, 2200, 1200), (2, 2100, 32777), (20, 2200, 700),
        (18, 700, 900), (30, 1400, 600), (25, 2000, 500), (40, 1400, 300), (60, 2010, 333)]


@pytest.mark.parametrize("dtype", base.DTYPES)
@pytest.mark.parametrize("rows,n", SIZES)
def test_quantize(rows, n, dtype):
    base.test_quantize(rows, n, dtype)


@pytest.mark.parametrize("dtype", base.DTYPES)
@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("add", [False, True])
def test_add_rmsnorm(rows, n, add, dtype):
    base.test_add_rmsnorm(rows, n, add, dtype)


@pytest.mark.parametrize("rows", [1, 140])
def test_the_longest_rows(rows):
    announce(f"longest rows {rows}")
    n, dtype = q8.MAX_IN, torch.bfloat16
    g = torch.Generator().manual_seed(rows)
    x, y = base.rows_of(g, dtype, rows, n), base.rows_of(g, dtype, rows, n)
    w = (1 + 0.2 * torch.randn(n, generator=g)).to(dtype)
    base.check_rows(q8.quantize(x.to(DEV)), x, 2 * base.U)
    r = o8.add(x, y)
    xd = x.to(DEV)
    res, got = q8.add_rmsnorm(xd, w.to(DEV), 1e-6, y=y.to(DEV), residual_out=xd)
    assert res is xd and torch.equal(res.cpu(), r)
    base.check_rows(got, o8.rmsnorm(r, w, 1e-6), LONGEST)


@pytest.mark.parametrize("dtype", base.DTYPES)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(m, n, k, dtype):
    base.test_product(m, n, k, dtype)


@pytest.mark.parametrize("dtype", base.DTYPES)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_linear_is_the_product_of_its_rows(m, n, k, dtype):
    base.test_linear_is_the_product_of_its_rows(m, n, k, dtype)


@pytest.mark.parametrize("dtype", base.DTYPES)
@pytest.mark.parametrize("m,hidden,inter", MLPS)
def test_mlp(m, hidden, inter, dtype):
    base.test_mlp(m, hidden, inter, dtype)
