"""The rule that chooses an 8-bit product's kernel (csrc/q8_rule.h), on the CPU: the measured winners, work-groups
that cover every result, and GPU tests that reach every kernel."""
import ctypes
import functools
import tempfile
from pathlib import Path

import pytest

import test_q8_gpu
from host_rules import rules

FEW, T32X32, T32X64, T64X64, G64, G128, G128X192, G192X128, G128X256, G192X192, G256X256 = range(11)
SHAPE = {T32X32: (32, 32), T32X64: (32, 64), T64X64: (64, 64), G64: (64, 64), G128: (128, 128),
         G128X192: (128, 192), G192X128: (192, 128), G128X256: (128, 256), G192X192: (192, 192),
         G256X256: (256, 256)}


@functools.lru_cache(None)
def _library():
    with tempfile.TemporaryDirectory() as tmp:
        fn = rules(Path(tmp), "q8_rule.h", """
int plan(int rows, int panels, int kp, int* tiles) {
  const mi_fa2::Q8Plan p = mi_fa2::q8_plan(rows, panels, kp);
  *tiles = p.tiles;
  return p.kernel;
}
int rows_shape(int panels, int kp) {
  const mi_fa2::Q8RowsShape s = mi_fa2::q8_rows_shape(panels, kp, 256);
  return 10 * s.panels + s.per_cu;
}""")
    fn.plan.argtypes = [ctypes.c_int] * 3 + [ctypes.POINTER(ctypes.c_int)]
    return fn


def plan(rows, features, k):
    tiles = ctypes.c_int()
    kernel = _library().plan(rows, -(-features // 16), -(-k // 128) * 128, ctypes.byref(tiles))
    return kernel, tiles.value


@pytest.mark.parametrize("rows,features,k,kernel", [
    (1, 2048, 1536, FEW), (16, 151936, 1536, FEW), (16, 100000, 8960, FEW), (17, 2048, 1536, FEW),
    (64, 6144, 2048, FEW), (32, 1536, 8960, FEW), (32, 6144, 4096, T32X32), (32, 14336, 4096, T32X64),
    (33, 1536, 8960, T32X32), (64, 6144, 4096, T32X64), (64, 9728, 896, G64), (64, 17920, 1536, G64),
    (17, 151936, 1536, G128), (150, 896, 4864, T32X32), (256, 1536, 8960, T32X64),
    (512, 1536, 8960, T64X64), (400, 2048, 1536, G64), (512, 17920, 1536, G192X128),
    (4096, 2048, 1536, G128), (2048, 17920, 1536, G128X192), (4001, 1536, 8960, G192X128), (4096, 1536, 8960, G128X192),
    (16384, 1536, 8960, G128X256), (6001, 6144, 4096, G192X192), (3000, 4096, 14336, G192X128),
    (8192, 8192, 8192, G256X256), (4096, 6144, 4096, G128X256), (1, 1, 1, FEW), (65, 1, 1, T32X32)])
def test_kernels(rows, features, k, kernel):
    assert plan(rows, features, k)[0] == kernel


def test_work_groups_cover_every_result():
    for rows in (1, 16, 17, 64, 65, 127, 129, 1000, 1 << 21):
        for features in (1, 16, 17, 1000, 17920):
            for k in (1, 2048, 2049, 131072):
                kernel, tiles = plan(rows, features, k)
                if kernel == FEW:
                    assert rows <= 64 and (k <= 2048 or rows <= 32)
                else:
                    tm, tn = SHAPE[kernel]
                    assert tiles == -(-rows // tm) * -(-features // tn)


def test_the_gpu_tests_reach_every_kernel():
    assert {plan(*size)[0] for size in test_q8_gpu.PRODUCTS} == set(range(11))
    assert {plan(m, 2 * inter, hidden)[0] for m, hidden, inter in test_q8_gpu.MLPS} == set(range(11))


def rows_shape(features, k):
    return divmod(_library().rows_shape(-(-features // 16), -(-k // 128) * 128), 10)


@pytest.mark.parametrize("features,k,shape", [
    (16, 16, (1, 1)), (4096, 2048, (1, 1)), (6720, 1536, (2, 1)), (9728, 896, (4, 1)), (17920, 1536, (2, 2)),
    (28672, 896, (4, 1)), (28672, 1536, (2, 2)), (22016, 2048, (2, 1)), (151936, 1536, (4, 1)), (151936, 2048, (2, 1))])
def test_few_rows(features, k, shape):
    assert rows_shape(features, k) == shape


def test_the_gpu_tests_reach_every_shape_of_few_rows():
    every = {((1, 1), 2), ((1, 1), 3), ((1, 1), 4), ((2, 1), 2), ((2, 1), 3), ((2, 1), 4), ((2, 2), 3), ((4, 1), 2),
             ((4, 1), 3)}
    steps = lambda k: max(2, -(-(-(-k // 128) * 128) // 512))
    assert {(rows_shape(n, k), steps(k)) for m, n, k in test_q8_gpu.PRODUCTS if m <= 16 and k <= 2048} == every
