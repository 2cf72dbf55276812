"""Workspaces of the operators that train a head hold what their kernels use, no more (host calls; no GPU)."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def so():
    from mace_onegpu import _lib
    return _lib.lib()


P, ONE = ctypes.c_void_p(0), ctypes.c_void_p(16)


def test_cross_entropy_partial_sums_by_the_tiles_taken(so):
    """Two floats a row and tile: 98,304 rows by 131,072 classes take tiles of 256, 403 MB and not 1.6 GB of 64."""
    n = ctypes.c_size_t(0)
    T, D, V = 98304, 64, 131072
    assert so.mm_ce_workspace(T, D, V, 1, ONE, 0, 0, ctypes.byref(n)) == 0
    packed = 2 * T * D
    assert T * V // 256 * 8 <= n.value - packed <= T * V // 256 * 8 + 2 ** 21
    # few tiles: of 64
    assert so.mm_ce_workspace(300, 64, 640, 1, ONE, 0, 0, ctypes.byref(n)) == 0
    assert 10 * 300 * 8 <= n.value - 2 * 300 * 64 <= 10 * 300 * 8 + 2 ** 14
