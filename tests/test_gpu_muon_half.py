"""Muon on float16 parameters: the update does not depend on the gradients' scale, so neither does it overflow nor vanish.

Gradients that float16 holds exactly, so a float32 twin with the same gradients has the same momentum and the same update;
the parameters differ by the float16 one's rounding, half a unit (2^-11 of the value, 2^-25 at least) a step."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("scale", [4000.0, 1.0, 2.0 ** -20])
def test_scale_of_half_gradients(scale, nesterov):
    from mace_onegpu.muon import Muon
    g = torch.Generator().manual_seed(1)
    steady = torch.randn(3, 24, 40, generator=g).clamp(-4, 4)
    p = [torch.nn.Parameter(torch.zeros(3, 24, 40, dtype=t, device="cuda")) for t in (torch.float16, torch.float32)]
    opt = Muon(p, lr=0.01, nesterov=nesterov)
    slack = torch.zeros(3, 24, 40, device="cuda")
    for step in range(45):
        grad = (scale * (steady + 0.1 * torch.randn(3, 24, 40, generator=g))).half()
        assert grad.isfinite().all()
        p[0].grad, p[1].grad = grad.cuda(), grad.cuda().float()
        opt.step()
        now = p[0].detach().float()
        slack += 2.0 ** -11 * now.abs() + 2.0 ** -25 + 2.0 ** -22 * now.abs()
        assert now.isfinite().all(), step
        assert bool(((now - p[1].detach()).abs() <= slack).all()), step
