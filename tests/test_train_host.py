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


def _ce(so, T=8, D=32, V=10, dtype=0, reduction=0, ldx=32, x=ONE, ws=ONE, w=ONE):
    return so.mm_ce_fwd(x, ldx, dtype, T, D, w, V, ONE, 0, -100, reduction, ONE, ONE, ONE, ws, P)


def test_cross_entropy_arguments(so):
    for bad in (dict(T=-1), dict(D=0), dict(V=0), dict(dtype=3), dict(reduction=3), dict(reduction=-1), dict(ldx=-1),
                dict(x=P), dict(ws=P), dict(w=P)):
        assert _ce(so, **bad) == -1, bad
    for far in (dict(T=2 ** 31 - 1), dict(V=2 ** 31 - 1), dict(D=2 ** 31 - 1), dict(T=10 ** 6, V=10 ** 6),
                dict(D=2 ** 17, V=2 ** 20)):
        assert _ce(so, **far) == -3, far
    args = [ONE, 32, 0, 8, 32, ONE, 10, 0, ONE, ONE, ONE, ONE, ONE, ONE, P]
    for i, v in ((2, 5), (3, 0), (4, 0), (6, 0), (7, 3), (8, P), (9, P), (10, P), (13, P)):
        assert so.mm_ce_bwd(*[v if q == i else a for q, a in enumerate(args)]) == -1, i
    args[11] = args[12] = P
    assert so.mm_ce_bwd(*args) == 0        # nothing asked for


def test_cross_entropy_workspace(so):
    n = ctypes.c_size_t(0)
    sizes = []
    for dx, dw in ((0, 0), (1, 0), (0, 1), (1, 1)):
        assert so.mm_ce_workspace(8192, 2048, 131072, 1, ONE, dx, dw, ctypes.byref(n)) == 0
        sizes.append(n.value)
        assert 0 < n.value < 2 ** 30       # far below the logits' 2 GB
    assert sizes[3] > sizes[1] and sizes[3] > sizes[2]
    assert so.mm_ce_workspace(8, 32, 10, 0, ONE, 0, 0, P) == -1


def test_orthogonalize_arguments(so):
    c = (ctypes.c_float * 15)(*(3.0, -4.0, 2.0) * 5)
    n = ctypes.c_size_t(0)
    for args, rc in (((2, 8, 8, 3), -1), ((-1, 8, 8, 0), -1), ((2, 0, 8, 0), -1), ((2, 8, 0, 0), -1),
                     ((65536, 8, 8, 0), -3), ((1, 65537, 8, 0), -3), ((1, 8, 65537, 0), -3), ((65535, 2048, 2048, 0), -3), ((0, 8, 8, 0), 0)):
        assert so.mm_orthogonalize_workspace(*args, ctypes.byref(n)) == rc, args
        batch, rows, cols, dtype = args
        assert so.mm_orthogonalize(ONE, dtype, batch, rows, cols, 5, c, 0.0, ONE, ONE, P) == rc, args
    assert so.mm_orthogonalize_workspace(2, 8, 8, 0, P) == -1
    for bad in ((ONE, -1, c, 0.0, ONE, ONE), (ONE, 5, P, 0.0, ONE, ONE), (ONE, 5, c, -1.0, ONE, ONE),
                (P, 5, c, 0.0, ONE, ONE), (ONE, 5, c, 0.0, P, ONE), (ONE, 5, c, 0.0, ONE, P)):
        m, steps, co, eps, out, ws = bad
        assert so.mm_orthogonalize(m, 0, 2, 8, 8, steps, co, eps, out, ws, P) == -1, bad
