"""Mixture, group norm, linear cross entropy and Muon together, as a fit uses them: gradients of a training step against
plain operations in 64 bits, the update against the iteration in 64 bits, a captured step, and the command."""
import pytest
import torch

pytestmark = pytest.mark.gpu

C3 = (3.4445, -4.7750, 2.0315)


def _parts(seed=1, atoms=300, classes=20):
    from mace_onegpu.expert_mix import ClassHead, ExpertMix
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(atoms, 4, 128, generator=g).cuda()
    y = torch.randint(0, classes, (atoms,), generator=g)
    y[torch.rand(atoms, generator=g) < 0.3] = -100
    return ExpertMix(n_experts=5, k=2), ClassHead(classes=classes), h, y.cuda()


def _plain(mix, head, h, y, sizes, params):
    """The loss in 64 bits with the module's choice of experts."""
    wn, bn, router, b0, b1, gw, gb, w = params
    s = h[:, 0]
    norm = (s - s.mean(1, keepdim=True)) / torch.sqrt(s.var(1, correction=0, keepdim=True) + 1e-5) * wn + bn
    e = mix.plan.experts.long()
    gates = torch.softmax((norm @ router).gather(1, e), 1)
    out = torch.cat([sum(gates[:, j, None, None] * torch.bmm(x, b[e[:, j]]) for j in range(2))
                     for x, b in ((h[:, :1], b0), (h[:, 1:], b1))], 1)
    x = out[:, 0] + out[:, 1:].square().sum(1)
    rows = []
    for part in x.split(sizes):
        v = part.view(part.shape[0], 8, 16)
        mu = v.mean((0, 2), keepdim=True)
        n = ((v - mu) / torch.sqrt(((v - mu) ** 2).mean((0, 2), keepdim=True) + 1e-5)).view(-1, 128)
        rows.append(torch.nn.functional.silu(n * gw + gb))
    return torch.nn.functional.cross_entropy(torch.cat(rows) @ w.T, y, ignore_index=-100)


@pytest.mark.parametrize("offsets", [None, [0, 120, 121, 300]])
def test_gradients_of_a_training_step(offsets):
    """Errors of the gates and products (as for the mixture alone), and of the norm's and the logits' sums of 128 to 4800
    terms, below 2e-4 of each result's largest value."""
    mix, head, h, y = _parts()
    params = [*mix.parameters(), *head.parameters()]
    assert [tuple(p.shape) for p in params] == [(128, 5), (128,), (128,), (5, 128, 128), (5, 128, 128), (20, 128),
                                                (128,), (128,)]
    router, wn, bn, b0, b1, w, gw, gb = params
    o = None if offsets is None else torch.tensor(offsets).cuda()
    loss = head(mix(h), y, o)
    grads = torch.autograd.grad(loss, params)
    d = [t.detach().double().requires_grad_() for t in (wn, bn, router, b0, b1, gw, gb, w)]
    sizes = [300] if offsets is None else [120, 1, 179]
    want = _plain(mix, head, h.double(), y, sizes, d)
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-4
    ref = dict(zip(("wn", "bn", "router", "b0", "b1", "gw", "gb", "w"), torch.autograd.grad(want, d)))
    for got, name in zip(grads, ("router", "wn", "bn", "b0", "b1", "w", "gw", "gb")):
        err, top = float((got.double() - ref[name]).abs().max()), float(ref[name].abs().max())
        assert err < 2e-4 * top, (name, err, top)


def test_update_by_muon():
    """A step on the gradients of the blocks and the head against the iteration in 64 bits."""
    from mace_onegpu.muon import Muon
    mix, head, h, y = _parts(2)
    params = [mix.router, *mix.blocks, head.weight]
    before = [p.detach().clone() for p in params]
    opt = Muon(params, lr=0.01, momentum=0.9)
    head(mix(h), y).backward()
    opt.step()
    for p, old in zip(params, before):
        u = 1.9 * p.grad.double().reshape(-1, *p.shape[-2:])       # grad + 0.9 buf, buf = grad in the first step
        x = u / (torch.linalg.matrix_norm(u)[:, None, None] + 1e-7)
        for _ in range(5):
            A = x @ x.mT.contiguous()
            x = C3[0] * x + (C3[1] * A + C3[2] * A @ A) @ x
        want = old.double() - 0.01 * 0.2 * max(p.shape[-2:]) ** 0.5 * x.view(p.shape)
        # the smallest singular values of a gradient of few atoms grow by 485 with their rounding
        assert float((p.detach().double() - want).abs().max()) < 1e-5


def test_captured_step():
    """Forward, backward and update in one graph, replayed on other atoms, against the same steps without it."""
    from mace_onegpu.muon import Muon

    def build():
        mix, head, h, y = _parts(3)
        params = [*mix.parameters(), *head.parameters()]
        opt = Muon([p for p in params if p.dim() >= 2], lr=0.01)

        def step():
            loss = head(mix(h), y)
            for p, g in zip(params, torch.autograd.grad(loss, params)):
                p.grad.copy_(g)
            opt.step()
            return loss.detach()

        for p in params:
            p.grad = torch.zeros_like(p)
        return h, y, params, step

    runs = [build(), build()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):                       # the optimizer's state exists before the capture
            for h, y, params, step in runs:
                step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = runs[0][3]()
    for seed in (4, 5, 6):
        _, _, h, y = _parts(seed)
        for run in runs:
            run[0].copy_(h)
            run[1].copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, runs[1][3]())
        for p, q in zip(runs[0][2], runs[1][2]):
            assert torch.equal(p, q)


def test_classes_of_equal_size():
    from mace_onegpu.expert_mix import equal_classes
    v = torch.randn(1001, generator=torch.Generator().manual_seed(7)).cuda()
    c = equal_classes(v, 10)
    assert c.min() == 0 and c.max() == 9 and int(torch.bincount(c).max()) - int(torch.bincount(c).min()) <= 1
    for k in range(9):
        assert float(v[c == k].max()) <= float(v[c == k + 1].min())


@pytest.mark.parametrize("extra", [["--bins", "16"], ["--bins", "16", "--muon"], ["--muon"]])
def test_command_runs(extra):
    from mace_onegpu.expert_mix import main
    res = main(["--water", "64", "--steps", "4", *extra])
    assert res["atoms"] == 192 and len(res["losses"]) == 4 and res["single"] < 1e-4
    assert all(v == v for v in res["losses"]) and ("--bins" not in extra or 0 <= res["right"] <= 1)
