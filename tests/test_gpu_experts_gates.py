"""expert_linear's gradients where the gates are not contiguous, for every set of inputs that ask for one, on each path.

Against 64 bits with the tolerances of test_gpu_experts.py (sums of n float32 products, (n + 16) 2^-24 of the
magnitudes, and the rounding of the output's type)."""
import itertools

import pytest
import torch
from test_gpu_experts import DTYPES, _check, _make, _reference

pytestmark = pytest.mark.gpu


def _column_slice(g):
    return torch.cat([g, torch.full_like(g, 9.0)], 1).cuda().requires_grad_()[:, :g.shape[1]]


def _transpose(g):
    return g.T.contiguous().cuda().requires_grad_().T


LAYOUTS = [_column_slice, _transpose]


def _every_subset(layout, T, M, D, F, E, k, dtype):
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, experts, gates, dy = _make(T, M, D, F, E, k, dtype, T + D + k, closed=0.05)
    ref, mag = _reference(x, w, experts, gates, dy)
    counts = int(torch.bincount(experts.clamp(min=0).reshape(-1).long()).max())
    terms = dict(y=D, dx=F, dg=F + M * D, dw=counts * M)
    names = ("dx", "dw", "dg")
    for want in itertools.product([False, True], repeat=3):
        if not any(want):
            continue
        xg, wg, gg = x.cuda().requires_grad_(want[0]), w.cuda().requires_grad_(want[1]), layout(gates)
        if not want[2]:
            gg = gg.detach()
        assert gg.requires_grad == want[2] and (k == 1 or not gg.is_contiguous())
        plan = plan_experts(experts.cuda(), E)                       # lists of this call alone
        y = expert_linear(xg, wg, plan, gg)
        inputs = [t for t, q in zip((xg, wg, gg), want) if q]
        got = torch.autograd.grad(y, inputs, dy.cuda())
        _check(dict(y=y, **dict(zip([n for n, q in zip(names, want) if q], got))), ref, mag, terms, dtype)


# few rows; slots; one choice joined, up to 128 columns and beyond; pairs held; pairs in tiles (16 bits); slots of pairs
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,M,D,F,E,k", [(5, 1, 64, 48, 4, 2), (900, 1, 72, 200, 5, 3), (700, 1, 64, 96, 4, 1),
                                         (700, 2, 264, 136, 3, 1), (9000, 1, 128, 256, 3, 2), (3000, 3, 160, 128, 2, 2)])
def test_strided_gates(T, M, D, F, E, k, dtype, layout):
    _every_subset(layout, T, M, D, F, E, k, dtype)


def test_pairs_of_16_bits():
    """Enough results for two choices in 16 bits to be joined in dx (16 M), with the gates' gradient asked or not."""
    _every_subset(_column_slice, 70000, 1, 256, 64, 3, 2, torch.bfloat16)


def test_expanded_gates():
    """One gate for both choices of a row: the gradient of an expanded tensor is the sum over its uses."""
    from mace_onegpu.experts import expert_linear, plan_experts
    for T in (4, 600):
        x, w, experts, gates, dy = _make(T, 1, 64, 48, 4, 2, torch.float32, T)
        gates = gates[:, :1].clone()
        ref, mag = _reference(x, w, experts, gates.expand(T, 2), dy)
        one = gates.cuda().requires_grad_()
        y = expert_linear(x.cuda(), w.cuda(), plan_experts(experts.cuda(), 4), one.expand(T, 2))
        (dg,) = torch.autograd.grad(y, one, dy.cuda())
        for d in (ref, mag):
            d["dg"] = d["dg"].sum(1, keepdim=True)
        _check(dict(y=y, dg=dg), ref, mag, dict(y=64, dg=48 + 64 + 1), torch.float32)


def test_gates_frozen_between_forward_and_backward():
    """Backward follows what forward saw, whatever requires_grad says by then."""
    from mace_onegpu.experts import expert_linear, plan_experts
    for T, D, F, E, k in ((9000, 128, 256, 3, 2), (700, 264, 136, 3, 1), (400, 64, 48, 4, 3)):
        x, w, experts, gates, dy = _make(T, 1, D, F, E, k, torch.float32, T)
        ref, mag = _reference(x, w, experts, gates, dy)
        for first in (True, False):
            xg, gg = x.cuda().requires_grad_(), gates.cuda().requires_grad_(first)
            y = expert_linear(xg, w.cuda(), plan_experts(experts.cuda(), E), gg)
            gg.requires_grad_(not first)
            (dx,) = torch.autograd.grad(y, xg, dy.cuda())
            _check(dict(dx=dx), ref, mag, dict(dx=F), torch.float32)
