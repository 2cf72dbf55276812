"""Refusals of the layer norm, routing and expert entry points, on the host before any launch (no GPU): the C ABI with
pointers that are never read, and the Python functions with CPU tensors.  Work of no rows is accepted."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "mace-million_amd", "lib", "libmace_million_amd.so")
needs_lib = pytest.mark.skipif(not os.path.exists(LIB), reason="library not built (python mace-million_amd/build.py)")
P, N = ctypes.c_void_p(0x1000), ctypes.c_void_p(0)


def _refused(name, args, code, match):
    from mace_onegpu import _lib
    assert getattr(_lib.lib(), name)(*args) == code
    assert match in _lib.last_error() and name in _lib.last_error()


def _with(base, **kw):
    return list(dict(base, **kw).values())


NORM = dict(x=P, ldx=64, dtype=0, rows=4, D=64, w=P, b=P, p_dtype=0, eps=1e-5, y=P, ldy=64, mean=N, rstd=N, stream=N)
NORM_BWD = dict(dy=P, lddy=64, x=P, ldx=64, dtype=0, rows=4, D=64, w=P, p_dtype=0, mean=P, rstd=P, dx=P, lddx=64, dw=P,
                db=P, workspace=P, stream=N)
ROUTE = dict(logits=P, ldl=8, dtype=0, T=4, E=8, k=2, scoring=0, bias=N, groups=1, top_groups=1, renorm=1, scale=1.0,
             gates=P, experts=P, stream=N)
ROUTE_BWD = dict(logits=P, ldl=8, dtype=0, T=4, E=8, k=2, scoring=0, renorm=1, scale=1.0, gates=P, experts=P, dgates=P,
                 dlogits=P, stream=N)
PLAN = dict(experts=P, S=8, E=4, offsets=P, order=P, scratch=N, stream=N)


@needs_lib
@pytest.mark.parametrize("change,code,match", [
    (dict(dtype=3), -1, "dtype"), (dict(dtype=-1), -1, "dtype"), (dict(dtype=0, p_dtype=1), -1, "weight and bias"),
    (dict(dtype=1, p_dtype=2), -1, "weight and bias"), (dict(D=0), -1, "sizes"), (dict(rows=-1), -1, "sizes"),
    (dict(ldx=-1), -1, "sizes"), (dict(ldy=63), -1, "sizes"), (dict(mean=P), -1, "together"),
    (dict(D=16385, ldx=16385, ldy=16385), -3, "16384")])
def test_layernorm_fwd(change, code, match):
    _refused("mm_layernorm_fwd", _with(NORM, **change), code, match)


@needs_lib
@pytest.mark.parametrize("change,code,match", [
    (dict(dtype=7), -1, "dtype"), (dict(p_dtype=2), -1, "weight and bias"), (dict(lddx=1), -1, "sizes"),
    (dict(workspace=N), -1, "workspace"), (dict(D=20000, lddx=20000), -3, "16384")])
def test_layernorm_bwd(change, code, match):
    _refused("mm_layernorm_bwd", _with(NORM_BWD, **change), code, match)


@needs_lib
@pytest.mark.parametrize("change,code,match", [
    (dict(dtype=5), -1, "dtype"), (dict(T=-1), -1, "sizes"), (dict(E=0), -1, "sizes"), (dict(k=0), -1, "sizes"),
    (dict(k=9), -1, "sizes"), (dict(ldl=7), -1, "sizes"), (dict(scoring=2), -1, "scoring"),
    (dict(groups=3), -1, "groups"),
    (dict(groups=4, top_groups=5), -1, "groups"), (dict(groups=4, top_groups=0), -1, "groups"),
    (dict(scale=0.0), -1, "scale"), (dict(E=1025, ldl=1025), -3, "1024"), (dict(E=64, ldl=64, k=33), -3, "32"),
    (dict(E=130, ldl=130, groups=65), -3, "64")])
def test_route(change, code, match):
    _refused("mm_route_fwd", _with(ROUTE, **change), code, match)
    if not set(change) & {"groups", "top_groups"}:
        _refused("mm_route_bwd", _with(ROUTE_BWD, **change), code, match)


@needs_lib
@pytest.mark.parametrize("change,code,match", [(dict(S=-1), -1, "sizes"), (dict(E=0), -1, "sizes"),
                                               (dict(E=1025), -3, "1024"), (dict(S=1000000), -1, "scratch")])
def test_plan(change, code, match):
    _refused("mm_expert_plan", _with(PLAN, **change), code, match)


@needs_lib
def test_no_rows_is_no_launch():
    from mace_onegpu import _lib
    so = _lib.lib()
    assert so.mm_layernorm_fwd(*_with(NORM, rows=0)) == 0
    assert so.mm_route_fwd(*_with(ROUTE, T=0)) == 0 and so.mm_route_bwd(*_with(ROUTE_BWD, T=0)) == 0


@needs_lib
def test_scratch_sizes():
    from mace_onegpu import _lib
    so = _lib.lib()
    n = ctypes.c_long(-1)
    assert so.mm_expert_plan_scratch(4096, 1024, ctypes.byref(n)) == 0 and n.value == 0      # one launch
    for S, E in ((20481, 1), (50000, 513), (2 ** 31 - 1, 1024)):                              # counts of every tile
        assert so.mm_expert_plan_scratch(S, E, ctypes.byref(n)) == 0 and n.value >= E * ((S + 4095) // 4096)
    assert so.mm_expert_plan_scratch(-1, 4, ctypes.byref(n)) == -1
    b = ctypes.c_size_t(0)
    assert so.mm_layernorm_workspace(0, 64, 0, ctypes.byref(b)) == 0 and b.value == 0
    assert so.mm_layernorm_workspace(10 ** 7, 64, 0, ctypes.byref(b)) == 0 and b.value % (2 * 64 * 4) == 0
    assert so.mm_layernorm_workspace(4, 16385, 0, ctypes.byref(b)) == -1


def test_cpu_tensors_are_refused():
    from mace_onegpu.experts import expert_linear, plan_experts, route
    from mace_onegpu.layer_norm import layer_norm
    x = torch.zeros(4, 8)
    e = torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: layer_norm(x), lambda: route(x, 2), lambda: plan_experts(e, 8),
                 lambda: expert_linear(x, torch.zeros(8, 8, 8), None)):
        with pytest.raises(TypeError, match="GPU tensor"):
            call()
