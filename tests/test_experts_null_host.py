"""Null pointers that the experts' entry points refuse on the host, before any launch (no GPU needed)."""
import ctypes
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "mace-million_amd", "lib", "libmace_million_amd.so")
pytestmark = pytest.mark.skipif(not os.path.exists(LIB), reason="library not built (python mace-million_amd/build.py)")
P, N = ctypes.c_void_p(0x1000), ctypes.c_void_p(0)

ROWS = {"in": P, "st": 8, "sm": 8, "dtype": 0, "S": 8, "k": 2, "M": 1, "K": 8, "N": 8, "W": P, "transposed": 0, "E": 4,
        "offsets": P, "order": P, "out": P, "stream": N}
JOINED = {"in": P, "st": 8, "sm": 8, "dtype": 0, "T": 4, "k": 1, "M": 1, "K": 8, "N": 8, "W": P, "transposed": 1, "E": 4,
          "gates": P, "experts": P, "offsets": P, "order": P, "out": P, "x": P, "xt": 8, "xm": 8, "dgates": N, "stream": N}
FEW = {"x": P, "st": 8, "sm": 8, "dtype": 0, "T": 4, "k": 2, "M": 1, "D": 8, "F": 8, "W": P, "E": 4, "gates": P,
       "experts": P, "y": P, "stream": N}
COMBINE = {"rows": P, "gates": P, "experts": P, "dtype": 0, "T": 4, "k": 2, "M": 1, "N": 8, "E": 4, "y": P, "stream": N}
COMBINE_BWD = {"rows": P, "gates": P, "experts": P, "x": P, "st": 8, "sm": 8, "dtype": 0, "T": 4, "k": 2, "M": 1, "N": 8,
               "E": 4, "dx": P, "dgates": P, "stream": N}
WGRAD = {"x": P, "xt": 8, "xm": 8, "dy": P, "yt": 8, "ym": 8, "dtype": 0, "S": 8, "k": 2, "M": 1, "D": 8, "F": 8, "E": 4,
         "gates": P, "offsets": P, "order": P, "dW": P, "workspace": N, "stream": N}


@pytest.mark.parametrize("name,base,which", [
    ("mm_expert_rows", ROWS, ("in", "W", "offsets", "order", "out")),
    ("mm_expert_joined", JOINED, ("in", "W", "experts", "offsets", "order")),
    ("mm_expert_few", FEW, ("x", "W", "experts", "y")),
    ("mm_expert_combine", COMBINE, ("rows", "experts", "y")),
    ("mm_expert_combine_bwd", COMBINE_BWD, ("rows", "experts", "x")),
    ("mm_expert_wgrad", WGRAD, ("x", "dy", "offsets", "order", "dW"))])
def test_null_pointers(name, base, which):
    from mace_onegpu import _lib
    for p in which:
        assert getattr(_lib.lib(), name)(*dict(base, **{p: N}).values()) == -1, p
        assert "null" in _lib.last_error() and name in _lib.last_error()


def test_no_rows_need_no_pointers():
    from mace_onegpu import _lib
    so = _lib.lib()
    nothing = dict(W=N, offsets=N, order=N, experts=N)
    for name, base, rows in (("mm_expert_rows", ROWS, "S"), ("mm_expert_joined", JOINED, "T"), ("mm_expert_few", FEW, "T"),
                             ("mm_expert_combine", COMBINE, "T"), ("mm_expert_combine_bwd", COMBINE_BWD, "T")):
        args = dict(base, **{q: v for q, v in nothing.items() if q in base}, **{rows: 0})
        assert getattr(so, name)(*args.values()) == 0
