"""Losses and gradients of rows that are certain of their class, relative to the loss itself.

Entries are multiples of 1/32 up to 4 whose products and sums are exact, so logits have no errors in any type.  u = 2^-24:
an exponential of z is off by (4 + |z|) u, sums of them have at most 64 + V / 64 roundings, the logarithm and the
quotients add 8 u.  With rest = sum over the other classes of exp(l - l_target): loss = log(1 + rest), d of the target
-rest / (1 + rest), d of the others exp(l - l_target) / (1 + rest), each relative.  d is rounded to the type (float16,
scaled by 2^14: to 2^-39 at least); products and the rounding of the results as in test_gpu_cross_entropy.py."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(T, V, seed, D=16):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-16, 17, (V, D), generator=g) / 8.0
    y = torch.randint(0, V, (T,), generator=g)
    x = w[y] * 2.0 ** torch.randint(-2, 2, (T, 1), generator=g)
    return x, w, y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V", [(1, 40), (3, 89), (16, 500), (16, 40001), (17, 89), (300, 89), (1000, 3000),
                                 (20000, 89), (3000, 20000)])
def test_rows_certain_of_their_class(T, V, dtype):
    from mace_onegpu.cross_entropy import linear_cross_entropy
    x, w, y = (t.cuda() for t in _inputs(T, V, T + V))
    xd, wd = x.double(), w.double()
    z = xd @ wd.T.contiguous()
    z -= z.gather(1, y[:, None]).clone()
    e = torch.exp(z).scatter(1, y[:, None], 0.0)
    rest = e.sum(1, keepdim=True)
    want = torch.log1p(rest).squeeze(1)
    d = (e / (1 + rest)).scatter(1, y[:, None], -rest / (1 + rest))
    asked = z.abs().clamp_max(90)                            # those beyond vanish
    rel = U * (16 + 64 + V / 64) + U * (e * asked).sum(1) / rest.squeeze(1).clamp_min(1e-300)
    if T > 16:
        assert float(want.min()) < 1e-6 and bool((want > 0.1).any())
    xs, ws = x.to(dtype).requires_grad_(), w.to(dtype).requires_grad_()
    assert torch.equal(xs.detach().float(), x) and torch.equal(ws.detach().float(), w)
    loss = linear_cross_entropy(xs, ws, y, reduction="none")
    err = (loss.detach().double() - want).abs()
    bound = rel * want + U * want + 1e-37 * V
    assert bool((err <= bound).all()), float((err / bound).max())
    mean = linear_cross_entropy(xs, ws, y)
    assert abs(float(mean.detach().double()) - float(want.mean())) <= float(bound.mean() + 64 * U * want.mean())

    gx, gw = torch.autograd.grad(loss, (xs, ws), torch.ones_like(loss))
    P = 6 if dtype == torch.float32 else 1
    ad = d.abs()
    ed = ad * (2 * rel[:, None] + U * (16 + asked) + (4 * U if dtype == torch.float32 else HALF_ULP[dtype])) + 1e-37
    if dtype == torch.float16:
        ed = ed + 2.0 ** -39
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-36
    for got, ref, bound in [(gx, d @ wd, (ed + (P * V + 8) * U * ad) @ wd.abs()),
                            (gw, d.T.contiguous() @ xd, (ed + (P * T + 16) * U * ad).T.contiguous() @ xd.abs())]:
        bound = bound + HALF_ULP[dtype] * ref.abs() + tiny
        err = (got.double() - ref).abs()
        assert bool((err <= bound).all()), float((err / bound).max())


def test_losses_of_every_size():
    """One class beside the target, gap by gap: log(1 + exp(-gap)) down to the smallest normal float; exact ties."""
    from mace_onegpu.cross_entropy import linear_cross_entropy
    gap = torch.arange(0.0, 86.0, 0.25)
    x = torch.stack([gap, torch.zeros_like(gap)], 1).cuda()
    w = torch.tensor([[1.0, 0.0], [0.0, 1.0]]).cuda()
    y = torch.zeros(gap.numel(), dtype=torch.long).cuda()
    want = torch.log1p(torch.exp(-gap.double()))
    for T in (gap.numel(), 1):                     # by tiles, and a row at a time
        got = torch.cat([linear_cross_entropy(x[i:i + T], w, y[i:i + T], reduction="none")
                         for i in range(0, gap.numel(), T)]).double().cpu()
        assert bool(((got - want).abs() <= U * (24 + 2 * gap) * want).all()), float(((got - want).abs() / want).max())
