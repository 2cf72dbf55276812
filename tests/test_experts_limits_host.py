"""The largest sizes that the routing and expert entry points take, refused or sized on the host (no GPU, no memory)."""
import ctypes
import os

import pytest
from test_experts_host import ROUTE, ROUTE_BWD
from test_experts_null_host import COMBINE, COMBINE_BWD, FEW, JOINED, ROWS, WGRAD

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "mace-million_amd", "lib", "libmace_million_amd.so")
pytestmark = pytest.mark.skipif(not os.path.exists(LIB), reason="library not built (python mace-million_amd/build.py)")
MOST = 2 ** 31 - 2 ** 16


def _refused(name, args, match):
    from mace_onegpu import _lib
    assert getattr(_lib.lib(), name)(*args.values()) == -3
    assert match in _lib.last_error() and name in _lib.last_error()


@pytest.mark.parametrize("name,base,rows", [("mm_expert_rows", ROWS, "S"), ("mm_expert_joined", JOINED, "T"),
                                            ("mm_expert_wgrad", WGRAD, "S")])
def test_rows(name, base, rows):
    _refused(name, dict(base, **{rows: MOST + 1}), "2^31 - 2^16 rows")
    _refused(name, dict(base, **{rows: MOST // 3 + 1, "M": 3}), "2^31 - 2^16 rows")


def test_few_rows_of_many_columns():
    _refused("mm_expert_few", dict(FEW, F=2 ** 31 - 1), "too large for one launch")


@pytest.mark.parametrize("E,lanes", [(4, 4), (16, 4), (17, 8), (32, 8), (33, 16), (256, 16), (257, 32), (512, 32), (513, 64),
                                     (1024, 64)])
def test_routed_rows_are_threads_of_one_launch(E, lanes):
    rows = 2 ** 32 // lanes
    for name, base in (("mm_route_fwd", ROUTE), ("mm_route_bwd", ROUTE_BWD)):
        for T in (rows - 255, rows, 2 ** 33):
            _refused(name, dict(base, T=T, E=E, ldl=E), "too many rows")


@pytest.mark.parametrize("D,F,E", [(128, 128, 1), (65408, 1, 1), (1, 65408, 1), (128, 128, 511), (1024, 1024, 7)])
@pytest.mark.parametrize("S,M", [(MOST, 1), (MOST // 3, 3), (10 ** 9, 2)])
def test_partial_sums_of_the_longest_lists(S, M, D, F, E):
    """The chunks fill the card about once whatever the rows' number: never more partial sums than workgroups of two
    rounds (1024) and a cut chunk a list."""
    from mace_onegpu import _lib
    n = ctypes.c_size_t(0)
    assert _lib.lib().mm_expert_wgrad_workspace(S, M, D, F, E, ctypes.byref(n)) == 0
    assert D * F * 4 <= n.value <= (1024 + E) * D * F * 4
    assert _lib.lib().mm_expert_wgrad_workspace(MOST + 1, 1, D, F, E, ctypes.byref(n)) == -3


@pytest.mark.parametrize("name,base,widths", [
    ("mm_expert_rows", ROWS, "KN"), ("mm_expert_joined", JOINED, "KN"), ("mm_expert_few", FEW, "D"),
    ("mm_expert_combine", COMBINE, "N"), ("mm_expert_combine_bwd", COMBINE_BWD, "N"), ("mm_expert_wgrad", WGRAD, "DF")])
def test_widths(name, base, widths):
    """An index a tile past the last column still fits an int."""
    for w in widths:
        for n in (MOST + 1, 2 ** 31 - 1):
            _refused(name, dict(base, **{w: n}), "2^31 - 2^16 rows or columns")
