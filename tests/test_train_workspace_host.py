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


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_orthogonalize_in_one_workgroup(so, dtype):
    """Matrices that a workgroup holds through all steps take next to nothing; the call without the steps is for any."""
    n, whole = ctypes.c_size_t(0), ctypes.c_size_t(0)
    for batch, rows, cols in ((89, 201, 137), (1, 1, 1), (65535, 64, 64), (300, 128, 256)):
        assert so.mm_orthogonalize_workspace(batch, rows, cols, dtype, ctypes.byref(whole)) == 0
        for steps in (0, 5, 16):
            assert so.mm_orthogonalize_workspace_steps(batch, rows, cols, dtype, steps, ctypes.byref(n)) == 0
            assert 0 < n.value <= 256
        assert so.mm_orthogonalize_workspace_steps(batch, rows, cols, dtype, 17, ctypes.byref(n)) == 0
        assert n.value == whole.value > 256
    for batch, rows, cols in ((3, 513, 260), (1, 4096, 8192), (9, 300, 20)):
        assert so.mm_orthogonalize_workspace(batch, rows, cols, dtype, ctypes.byref(whole)) == 0
        assert so.mm_orthogonalize_workspace_steps(batch, rows, cols, dtype, 5, ctypes.byref(n)) == 0
        assert n.value == whole.value
    assert so.mm_orthogonalize_workspace_steps(0, 8, 8, dtype, 5, ctypes.byref(n)) == 0 and n.value == 0
    for args, rc in (((2, 8, 8, 3, 5), -1), ((-1, 8, 8, 0, 5), -1), ((2, 0, 8, 0, 5), -1), ((2, 8, 8, 0, -1), -1),
                     ((65536, 8, 8, 0, 5), -3), ((1, 65537, 8, 0, 5), -3)):
        assert so.mm_orthogonalize_workspace_steps(*args, ctypes.byref(n)) == rc, args
    assert so.mm_orthogonalize_workspace_steps(2, 8, 8, 0, 5, P) == -1
