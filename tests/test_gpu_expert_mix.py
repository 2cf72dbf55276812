"""ExpertMix: equivariance, its value and gradients against plain operations in 64 bits, and the command."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _mix(**kw):
    from mace_onegpu.expert_mix import ExpertMix
    return ExpertMix(**kw)


def test_value_and_gradients_against_plain_operations():
    """64-bit autograd through the same formula with the module's choice of experts.  Errors of the gates (96 u, and of
    the logits behind them: 128 products and a norm, 250 u of magnitudes below 40) and products (144 u) stay below
    1e-4 of each result's largest value."""
    m = _mix(n_experts=5, k=2)
    h = torch.randn(300, 4, 128, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    out = m(h)
    dy = torch.randn(out.shape, generator=torch.Generator().manual_seed(2)).cuda()
    params = [h, m.norm.weight, m.norm.bias, m.router, *m.blocks]
    grads = torch.autograd.grad(out, params, dy)
    hd, wn, bn, r, *blocks = (t.detach().double().requires_grad_() for t in params)
    s = hd[:, 0]
    norm = (s - s.mean(1, keepdim=True)) / torch.sqrt(s.var(1, correction=0, keepdim=True) + 1e-5) * wn + bn
    e = m.plan.experts.long()
    logits = norm @ r
    top = torch.sort(logits, dim=1, descending=True).values
    clear = (top[:, 1] - top[:, 2]) > 1e-4          # rows whose choice does not hang on a rounding
    assert torch.equal(logits.topk(2, 1).indices.sort(1).values[clear], e.sort(1).values[clear])
    gates = torch.softmax(logits.gather(1, e), 1)
    want = torch.cat([sum(gates[:, j, None, None] * torch.bmm(x, b[e[:, j]]) for j in range(2))
                      for x, b in ((hd[:, :1], blocks[0]), (hd[:, 1:], blocks[1]))], 1)
    assert float((out - want).detach().abs().max()) < 1e-4 * float(want.detach().abs().max())
    for got, ref in zip(grads, torch.autograd.grad(want, [hd, wn, bn, r, *blocks], dy.double())):
        assert float((got.double() - ref).abs().max()) < 1e-4 * float(ref.abs().max())


def test_rotations_of_the_vectors_commute():
    m = _mix(n_experts=4, k=2)
    h = torch.randn(500, 4, 128, generator=torch.Generator().manual_seed(3)).cuda()
    R = torch.linalg.qr(torch.randn(3, 3, generator=torch.Generator().manual_seed(4)))[0].cuda()
    turn = lambda x: torch.cat([x[:, :1], torch.einsum("ab,nbc->nac", R, x[:, 1:])], 1)  # noqa: E731
    with torch.no_grad():
        a, b = m(turn(h)), turn(m(h))
    assert float((a - b).abs().max()) < 1e-4 * float(b.abs().max())
    assert torch.equal(m(h.view(500, 512)), m(h))


def test_balance_evens_the_load():
    m = _mix(n_experts=8, k=2)
    h = torch.randn(2000, 4, 128, generator=torch.Generator().manual_seed(5)).cuda()
    h[:, 0] += 0.5                                   # a common direction: some experts are liked by most atoms
    with torch.no_grad():
        m.router += 0.05 * torch.randn(1, 8, generator=torch.Generator().manual_seed(6)).cuda()
        m(h)
        before = m.plan.counts.float().std()
        for _ in range(60):
            m(h)
            m.update_balance(2e-2)
        m(h)
    assert float(m.plan.counts.float().std()) < 0.5 * float(before) + 20
    with pytest.raises(ValueError, match="features must be"):
        m(h[:, :3])


def test_command_fits():
    from mace_onegpu.expert_mix import main
    res = main(["--water", "64", "--steps", "40"])
    assert res["atoms"] == 192 and res["losses"][-1] < 0.7 * res["losses"][0] and res["single"] < 1e-4
