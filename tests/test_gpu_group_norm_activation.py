"""The activations of group_norm and their slopes in float32, relative to themselves.

Weights of zero make the activation's argument the bias, so that it has no error: y = act(b), and db of one row is dy
times the slope there.  u = 2^-24: an exponential of an argument a is off by (2.5 |a| + 2) u, a = z^2 / 2 (gelu) or z (silu); a
reciprocal by 2 u, the normal distribution's tail by 10 u beside its exponential, products and sums by 8 u of their terms."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("offsets", [None, [0, 1]])
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_activation_and_slope(kind, offsets):
    from mace_onegpu.group_norm import group_norm
    z = torch.cat([torch.linspace(-11, 11, 3980), torch.tensor([0.0, -0.0, 1e-3, -1e-3, 1e-20, -1e-20, -3.0, -4.0, -5.0,
                                                                -6.0, -8.0, 3.0, 6.0, 40.0, 80.0, 1e4])])
    C = z.numel()
    x = torch.randn(1, 1, C, generator=torch.Generator().manual_seed(0)).cuda().requires_grad_()
    w, b = torch.zeros(C, device="cuda"), z.cuda().requires_grad_()
    if offsets is None:
        y = group_norm(x, 4, w, b, activation=kind)
    else:
        y = group_norm(x[0], 4, w, b, activation=kind, offsets=torch.tensor(offsets).cuda())
    db, = torch.autograd.grad(y.sum(), b)
    y, db, z = y.detach().double().cpu().view(C), db.double().cpu(), z.double()
    if kind == "silu":
        q, a = torch.sigmoid(z), z.abs()
        rel = U * (2.5 * a + 20)
        want, slope = z * q, q * (1 + z * (1 - q))
        eslope = rel * (q + (z * q * (1 - q)).abs()) + U * (z * q).abs()
    else:
        q, a = torch.special.erfc(-z / 2 ** 0.5) / 2, z * z / 2     # ndtr loses its tail
        rel = U * (2.5 * a + 22)
        bell = torch.exp(-a) * 0.3989422804014327
        want, slope = z * q, q + z * bell
        eslope = rel * (q + (z * bell).abs())
    err = (y - want).abs()
    assert bool((err <= rel * want.abs() + 1e-37).all()), float((err / want.abs().clamp_min(1e-30)).max())
    err = (db - slope).abs()
    assert bool((err <= eslope + 1e-37).all()), float((err / eslope.clamp_min(1e-30)).max())
