"""Dual tensors and traces are refused: the operators have no forward-mode derivative and are no dispatched operations, so
a tangent would vanish from the result and a trace would record nothing of them."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def _calls():
    from mace_onegpu.experts import expert_linear, plan_experts, route
    from mace_onegpu.layer_norm import layer_norm
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    experts = torch.randint(0, 4, (30, 2), generator=g).cuda()
    plan = plan_experts(experts, 4)
    yield "layer_norm", layer_norm, [r(30, 24), r(24), r(24)]
    yield "route", lambda x: route(x, 2)[0], [r(30, 8)]
    yield "expert_linear", lambda x, w, q: expert_linear(x, w, plan, q), [r(30, 24), r(4, 24, 16), r(30, 2)]


def test_dual_tensors():
    for name, f, args in _calls():
        for i in range(len(args)):
            for grad in (False, True):
                with fwAD.dual_level():
                    mixed = [fwAD.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t)) if q == i else t
                             for q, t in enumerate(args)]
                    with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
                        f(*mixed)
                    with torch.no_grad(), pytest.raises(RuntimeError, match=f"{name} has no forward-mode"):
                        f(*mixed)
                    assert f(*args).shape[0] == 30         # other tensors at the same time
                    plain = [fwAD.unpack_dual(t).primal.detach() for t in mixed]
                    assert torch.equal(f(*plain), f(*args))


def test_bias_of_the_choice_may_be_dual():
    """It moves the choice only and has no derivative."""
    from mace_onegpu.experts import route
    x, b = torch.randn(20, 8, generator=torch.Generator().manual_seed(1)).cuda(), torch.arange(8.0).cuda()
    with fwAD.dual_level():
        gates, experts = route(x, 2, bias=fwAD.make_dual(b, torch.ones_like(b)))
    want = route(x, 2, bias=b)
    assert torch.equal(gates, want[0]) and torch.equal(experts, want[1])


def test_traces():
    from mace_onegpu.experts import plan_experts
    for name, f, args in _calls():
        with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
            torch.jit.trace(f, tuple(args))
    with pytest.raises(RuntimeError, match="plan_experts cannot be traced"):
        torch.jit.trace(lambda e: plan_experts(e, 4).counts, (torch.zeros(3, 2, dtype=torch.int32, device="cuda"),))
