"""CPU: how the kernel for few rows is chosen, and that the GPU tests run every way of it."""

import ctypes
import random

import pytest

import dense_rows_shapes as rs
from easy_as_b200.runtime import cuda_ext


def test_gpu_tests_reach_every_way():
    """Plain and gated, by words, shifted and by values, 8 and 16 warps, K whole and shared."""
    covered = set().union(*(rs.ways(s) for s in rs.SHAPES))
    rng = random.Random(0)
    for _ in range(20000):
        m, n, k = rng.randint(1, 8), int(2 ** rng.uniform(0, 15)), int(2 ** rng.uniform(0, 15.3))
        if m * ((k + 63) // 64 * 128 + 64) > 81920:
            continue
        missing = rs.ways((m, n, k)) - covered
        assert not missing, ((m, n, k), missing)
    for gated in (False, True):
        for warps in (8, 16):
            for split in (1, 2):
                assert {(gated, way, warps, split) for way in (rs.WORDS, rs.SHIFTED)} <= covered
        assert {c[2:] for c in covered if c[0] == gated and c[1] == rs.VALUES} == {(8, 1), (8, 2)}


def test_plan_of_named_sizes():
    """x of up to 40960 bytes leaves room for two blocks per SM; less than half a tile per block shares K."""
    assert rs.plan(False, 1, 4096, 4096, False) == (rs.WORDS, 8, 1)
    assert rs.plan(False, 8, 300, 5000, False) == (rs.WORDS, 16, 1)    # x of 81408 bytes
    assert rs.plan(False, 8, 300, 5000, True) == (rs.VALUES, 8, 2)     # which values do not keep there
    assert rs.plan(False, 3, 600, 8203, True) == (rs.SHIFTED, 16, 2)
    assert rs.plan(True, 3, 600, 8203, True) == (rs.SHIFTED, 16, 1)
    assert rs.plan(False, 1, 1024, 8192, False) == (rs.WORDS, 8, 2)


@pytest.mark.parametrize("bad", [(2, 1, 8, 8), (-1, 1, 8, 8), (0, 0, 8, 8), (0, 9, 8, 8), (0, 1, 0, 8), (0, 8, 8, 8192)])
def test_plan_checks_its_arguments(bad):
    v = [ctypes.byref(ctypes.c_int()) for _ in range(3)]
    lib = cuda_ext.load()
    assert lib.eas_dense_rows_plan(*bad, 0, 148, *v) == cuda_ext.EAS_ERR_VALUE
    assert lib.eas_dense_rows_plan(0, 1, 8, 8, 0, 0, *v) == cuda_ext.EAS_ERR_VALUE
    assert lib.eas_dense_rows_plan(0, 1, 8, 8, 0, 148, None, v[0], v[1]) == cuda_ext.EAS_ERR_VALUE
