"""Which variant of the few-row kernel a product takes (q8_rows_choice in csrc/q8_rule.h), on the CPU: every one
that some size takes is taken by a size of the GPU tests."""
import ctypes
import functools
import itertools
import tempfile
from pathlib import Path

import pytest

import test_q8_gpu
import test_q8_wide_gpu
from host_rules import rules
from test_q8_rule import FEW, plan

PLAIN, NORM, FLOAT, ROWS = range(4)
CUS = 256


@functools.lru_cache(None)
def _library():
    with tempfile.TemporaryDirectory() as tmp:
        return rules(Path(tmp), "q8_rule.h", """
void choice(int rows, int panels, int kp, int cus, int source, int gated, int* out) {
  const mi_fa2::Q8RowsChoice c = mi_fa2::q8_rows_choice(rows, panels, kp, cus, (mi_fa2::Q8Source)source, gated);
  out[0] = c.mt, out[1] = c.panels, out[2] = c.half, out[3] = c.keep, out[4] = c.steps, out[5] = c.grid;
}""")


def pad(k):
    return -(-k // 128) * 128


def choice(source, gated, rows, panels, k):
    """(tokens by 16, panels of a tile, half, x kept, steps, grid)."""
    out = (ctypes.c_int * 6)()
    _library().choice(rows, panels, pad(k), CUS, source, gated, out)
    return tuple(out)


def variant(source, gated, rows, panels, k):
    """The kernel's template arguments."""
    return (source, gated, *choice(source, gated, rows, panels, k)[:5], source == FLOAT and rows == 1)


def fused(rows, k):
    return rows <= 16 and pad(k) <= 2048


def few(rows, panels, k):
    return plan(rows, panels * 16, k)[0] == FEW


def of_product(rows, n, k):
    """A product of rows in 8 bits, and of 16-bit rows with the norm and without."""
    panels = -(-n // 16)
    if few(rows, panels, k):
        yield variant(ROWS, False, rows, panels, k)
    if fused(rows, k):
        yield from (variant(s, False, rows, panels, k) for s in (PLAIN, NORM))


def of_mlp(rows, hidden, inter):
    first, second = -(-inter // 8), -(-hidden // 16)
    if fused(rows, hidden):
        yield from (variant(s, True, rows, first, hidden) for s in (PLAIN, NORM))
    elif few(rows, first, hidden):
        yield variant(ROWS, True, rows, first, hidden)
    if rows <= 4 and pad(inter) <= 12288:
        yield variant(FLOAT, False, rows, second, inter)
    elif few(rows, second, inter):
        yield variant(ROWS, False, rows, second, inter)


LENGTHS = (100, 1024, 1100, 1536, 1600, 2048, 2100, 4096, 9216, 12288, 12400, 131072)
WIDTHS = (1, 8, 100, 128, 129, 256, 257, 512, 513, 600, 1024, 1025, 2048, 2049, 4095, 4096, 9000, 70000)


def test_every_variant_is_run_on_the_gpu():
    every = set()
    for rows, k, panels in itertools.product((1, 2, 4, 5, 16, 17, 32, 33, 64), LENGTHS, WIDTHS):
        every.update(of_product(rows, 16 * panels, k))
        every.update(of_mlp(rows, k, 8 * panels))
        every.update(of_mlp(rows, 16 * panels, k))
    reached = set()
    for tests in (test_q8_gpu, test_q8_wide_gpu):
        for size in tests.PRODUCTS:
            reached.update(of_product(*size))
        for size in tests.MLPS:
            reached.update(of_mlp(*size))
    assert reached == every


@pytest.mark.parametrize("source,gated,rows,n,k,want", [
    # (measured winners: q8_rule.h)
    (NORM, False, 16, 6720, 1536, (1, 2, 0, 1, 3, 210)), (NORM, False, 1, 9728, 896, (1, 4, 0, 1, 2, 152)),
    (NORM, True, 1, 17920, 1536, (1, 2, 0, 1, 3, 512)), (ROWS, False, 16, 6400, 2048, (1, 1, 0, 1, 4, 256)),
    (ROWS, False, 64, 8192, 1536, (4, 1, 0, 1, 3, 256)), (FLOAT, False, 1, 1536, 8960, (1, 1, 1, 0, 18, 192)),
    (ROWS, False, 16, 1536, 8960, (1, 1, 1, 0, 9, 192)), (ROWS, False, 16, 100000, 4096, (1, 4, 0, 0, 9, 256)),
    (ROWS, False, 32, 1536, 8960, (2, 1, 0, 0, 6, 96)), (FLOAT, False, 4, 4096, 12288, (1, 1, 0, 0, 9, 256))])
def test_choices(source, gated, rows, n, k, want):
    assert choice(source, gated, rows, -(-n // 16), k) == want


def test_the_grid_is_never_more_than_the_tiles():
    for source, rows, k, panels in itertools.product(range(4), (1, 16, 17, 64), LENGTHS, WIDTHS):
        mt, np, half, _, _, grid = choice(source, False, rows, panels, k)
        assert 1 <= grid <= (2 * panels if half else -(-panels // np))
