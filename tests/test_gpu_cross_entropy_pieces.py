"""Losses whose gradients are taken in several pieces of the classes with the products' sums in parts, against the formula
in 64 bits, with the tolerances of test_gpu_cross_entropy.py."""
import pytest
import torch

from test_gpu_cross_entropy import _check, _inputs, _reference, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,D,V,dtype", [(3001, 77, 32003, torch.float16), (3001, 40, 32003, torch.bfloat16),
                                         (3001, 40, 30000, torch.float32), (9000, 64, 9000, torch.bfloat16)])
def test_pieces_with_split_sums(T, D, V, dtype):
    x, w, y, dloss = (t.cuda() for t in _inputs(T, D, V, dtype, T + V))
    ref, bound = _reference(x, w, y, dloss, "none", dtype)
    got = _run(x, w, y, dloss, "none")
    _check(got, ref, bound)
    again = _run(x, w, y, dloss, "none")
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("T,D,dtype", [(4, 256, torch.float32), (1, 513, torch.bfloat16)])
def test_few_rows_in_pieces(T, D, dtype):
    """More classes than a piece holds, by the kernel for few rows: every class's gradient, against 64 bits."""
    from mace_onegpu.cross_entropy import linear_cross_entropy
    V = 1100003
    g = torch.Generator(device="cuda").manual_seed(T)
    w = torch.randn(V, D, generator=g, device="cuda").mul_(2 / D ** 0.5).to(dtype).requires_grad_()
    x = torch.randn(T, D, generator=g, device="cuda").to(dtype).requires_grad_()
    y = torch.tensor([V - 1, 0, 600000, 7])[:T].cuda()
    loss = linear_cross_entropy(x, w, y, reduction="none")
    up = 0.5 + torch.rand(T, generator=g, device="cuda")
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    with torch.no_grad():
        logits = x.double() @ w.double().T
        lse = torch.logsumexp(logits, 1)
        assert float((loss.double() - (lse - logits[range(T), y])).abs().max()) < 1e-5
        d = torch.exp(logits - lse[:, None])
        d[range(T), y] -= 1
        d *= up.double()[:, None]
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
        # a lane sums D / 64 products of a logit and moves six times: off by (D / 64 + 6) 2^-24 sum |x w| < 3e-5, and so
        # is the log of the sum; exponentials down to -40: d is off by less than 1e-4 of itself, then rounded to the type;
        # sums as in test_gpu_cross_entropy.py
        e, P = 1e-4, 6 if dtype == torch.float32 else 1
        ref = d @ w.double()
        bound = (e + 2 * half + (P * V + 8) * 2.0 ** -24) * (d.abs() @ w.double().abs())
        assert bool(((dx.double() - ref).abs() <= bound + 1e-30).all())
        for i in range(0, V, 200000):
            p, a = d[:, i:i + 200000].T.contiguous(), x.double()
            err = (dw[i:i + 200000].double() - p @ a).abs()
            assert bool((err <= (e + 2 * half) * (p.abs() @ a.abs()) + 1e-30).all()), i
