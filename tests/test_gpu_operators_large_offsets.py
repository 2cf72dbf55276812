"""Rows whose offsets pass 2^32 elements: the last rows of a strided array give the same bits as a small copy of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TAIL = 300


def _wide(rows, comps, D):
    """float16 [rows, comps, D] beyond 2^32 elements, filled only where it is looked at"""
    x = torch.zeros(rows, comps, D, dtype=torch.float16, device="cuda")
    assert x.numel() > 2 ** 32
    x[-TAIL:] = torch.randn(TAIL, comps, D, generator=torch.Generator().manual_seed(1)).half().cuda()
    return x


def test_layer_norm():
    from mace_onegpu.layer_norm import layer_norm
    x = _wide(140000, 4, 8192)[:, 3].requires_grad_()
    w, b = (torch.randn(8192, generator=torch.Generator().manual_seed(s)).half().cuda().requires_grad_() for s in (2, 3))
    y = layer_norm(x, w, b)
    dy = torch.zeros_like(y)
    dy[-TAIL:] = 1.0
    (dx,) = torch.autograd.grad(y, x, dy)
    small = x.detach()[-TAIL:].clone().requires_grad_()
    z = layer_norm(small, w, b)
    (dz,) = torch.autograd.grad(z, small, dy[-TAIL:].clone())
    assert torch.equal(y[-TAIL:], z) and torch.equal(dx[-TAIL:], dz)


@pytest.mark.parametrize("k", [1, 2, 3])
def test_products(k):
    """dW of the zero rows is 0, so it is that of the last rows, up to the sums' order: two float32 sums of 300 terms."""
    from mace_onegpu.experts import expert_linear, plan_experts
    T = 1100000
    x = _wide(T, 4, 1024)[:, 1:].requires_grad_()                  # three components
    g = torch.Generator().manual_seed(k)
    w = (torch.randn(3, 1024, 24, generator=g) / 32).half().cuda().requires_grad_()
    e = torch.rand(T, 3, generator=g).topk(k, 1).indices.to(torch.int32).cuda()
    gates = torch.rand(T, k, generator=g).cuda().requires_grad_()
    y = expert_linear(x, w, plan_experts(e, 3), gates)
    assert not y[:-TAIL].any()
    dy = torch.randn(T, 1, 1, generator=g).half().cuda().expand(T, 3, 24)
    dw, dg = torch.autograd.grad(y, (w, gates), dy)
    small, gs = x.detach()[-TAIL:].clone(), gates.detach()[-TAIL:].clone().requires_grad_()
    ws = w.detach().clone().requires_grad_()
    z = expert_linear(small, ws, plan_experts(e[-TAIL:].clone(), 3), gs)
    dws, dgs = torch.autograd.grad(z, (ws, gs), dy[-TAIL:].clone())
    tol = dict(rtol=2.0 ** -10, atol=1e-3)                         # one unit of float16, and 1000 x 2^-24 x 24 below it
    assert torch.allclose(y[-TAIL:].float(), z.float(), **tol) and torch.allclose(dw.float(), dws.float(), **tol)
    assert not dg[:-TAIL].any() and torch.allclose(dg[-TAIL:], dgs, **tol)


def test_route():
    from mace_onegpu.experts import route
    wide = torch.zeros(4300000, 1024, dtype=torch.float16, device="cuda")
    assert wide.numel() > 2 ** 32
    wide[-TAIL:] = torch.randn(TAIL, 1024, generator=torch.Generator().manual_seed(4)).half().cuda()
    x = wide.requires_grad_()
    for kw in (dict(), dict(renormalize=False)):
        gates, experts = route(x, 4, **kw)
        (dx,) = torch.autograd.grad(gates[-TAIL:].square().sum(), x)
        small = x.detach()[-TAIL:].clone().requires_grad_()
        want, chosen = route(small, 4, **kw)
        (dz,) = torch.autograd.grad(want.square().sum(), small)
        assert torch.equal(gates[-TAIL:], want) and torch.equal(experts[-TAIL:], chosen) and torch.equal(dx[-TAIL:], dz)
