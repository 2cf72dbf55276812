"""Entry points of the operators that train a head refuse bad sizes before any launch (host calls on null or unused
pointers; no GPU)."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def so():
    from mace_onegpu import _lib
    return _lib.lib()


P = ctypes.c_void_p(0)
ONE = ctypes.c_void_p(16)   # a pointer that no refused call reads


def _norm(so, rows=8, structs=2, offsets=P, C=32, groups=4, dtype=0, p_dtype=0, act=0, ldx=32, ldy=32, ws=P, stats=P):
    return so.mm_groupnorm_fwd(ONE, ldx, dtype, rows, structs, offsets, C, groups, P, P, p_dtype, 1e-5, act, ONE, ldy,
                               stats, ws, P)


def test_group_norm_arguments(so):
    for bad in (dict(dtype=3), dict(dtype=-1), dict(p_dtype=2), dict(rows=-1), dict(structs=3), dict(C=0),
                dict(groups=5), dict(groups=0), dict(act=3), dict(act=-1), dict(ldy=31), dict(ldx=-1),
                dict(rows=2 ** 31 - 2 ** 16, structs=1), dict(offsets=ONE, structs=0),
                dict(rows=100000, structs=1)):     # tiles without the workspace
        assert _norm(so, **bad) == -1, bad
    assert _norm(so, C=4097, groups=1, ldx=4097, ldy=4097) == -3
    assert _norm(so, C=65536, groups=65536, ldx=65536, ldy=65536) == -3
    assert _norm(so, rows=0, structs=0) == 0
    assert so.mm_groupnorm_bwd(ONE, 32, ONE, 32, 0, 8, 2, P, 32, 4, P, P, 0, 0, ONE, ONE, 32, ONE, P, P, P) == -1
    assert so.mm_groupnorm_bwd(ONE, 32, ONE, 32, 0, 8, 2, P, 32, 4, P, P, 0, 3, ONE, ONE, 32, P, P, P, P) == -1


def test_group_norm_workspace(so):
    n = ctypes.c_size_t(123)
    assert so.mm_groupnorm_workspace(8, 2, 0, 32, 4, 0, 0, ctypes.byref(n)) == 0 and n.value == 0
    assert so.mm_groupnorm_workspace(8, 2, 0, 32, 4, 0, 1, ctypes.byref(n)) == 0 and n.value == 2 * 2 * 32 * 4
    assert so.mm_groupnorm_workspace(500000, 1, 0, 128, 8, 0, 0, ctypes.byref(n)) == 0 and n.value > 0
    assert so.mm_groupnorm_workspace(8, 3, 0, 32, 4, 0, 0, ctypes.byref(n)) == -1
    assert so.mm_groupnorm_workspace(8, 2, 0, 32, 4, 0, 0, P) == -1
