"""route and its gradient against a plain row-by-row implementation in 64 bits.

The choice is defined by float32 sums logit + bias and compared exactly.  Gates: u = 2^-24; an exponent's argument is a
difference rounded once (off by u |x - m|, |x - m| <= 40 here unless the exponential is 0 next to another), expf and
log1pf are good to 4 u, a sum of up to 1024 scores in lanes of 16 and trees has 26 roundings, and a division one more:
96 u in all, relative.  The gradient's terms carry the gates' errors and a sum over k <= 32 of them: 256 u of the sum
of magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _reference(logits, k, scoring, bias, groups, top_groups, renormalize, scale, dgates=None):
    """Row by row on the CPU: (gates, experts, dlogits, magnitude of dlogits' terms), 64 bits."""
    # the largest value first: -3.4e38 + log(n) is -3.4e38 in 64 bits as well
    normalised = lambda v: v - v.max() - torch.log(torch.exp(v - v.max()).sum())  # noqa: E731
    key32 = logits.float() if bias is None else logits.float() + bias.float()
    x = logits.double()
    T, E = x.shape
    gates, experts = torch.zeros(T, k, dtype=torch.float64), torch.full((T, k), -1, dtype=torch.int32)
    dl, mag = torch.zeros(T, E, dtype=torch.float64), torch.zeros(T, E, dtype=torch.float64)
    order = lambda v, idx: sorted(idx, key=lambda e: (0 if math.isnan(v[e]) else 1,  # noqa: E731
                                                      -v[e] if not math.isnan(v[e]) else 0.0, e))
    for t in range(T):
        keys = key32[t].tolist()
        row = x[t]
        closed = [bool(row[e] == -math.inf) or keys[e] == -math.inf for e in range(E)]
        keys = [-math.inf if c else v for c, v in zip(closed, keys)]
        gs = E // groups
        best = []
        for q in range(groups):
            first = order(keys, range(q * gs, (q + 1) * gs))[0]
            best.append(keys[first])
        open_ = set(order(best, range(groups))[:top_groups])
        cand = [e for e in order(keys, range(E)) if e // gs in open_ and keys[e] != -math.inf][:k]
        if not cand:
            continue
        e = torch.tensor(cand)
        logs = torch.nn.functional.logsigmoid(row) if scoring == "sigmoid" else normalised(row)
        l = logs[e]
        if renormalize:
            l = normalised(l)
        g = scale * torch.exp(l)
        gates[t, :len(cand)], experts[t, :len(cand)] = g, e.to(torch.int32)
        if dgates is None:
            continue
        d = dgates[t, :len(cand)].double()
        a = g * d
        m = a.abs()
        if renormalize:
            a, m = a - g / scale * (g * d).sum(), m + (g / scale).abs() * (g * d).abs().sum()
        s = torch.sigmoid(-row[e]) if scoring == "sigmoid" else torch.ones_like(a)
        dl[t, e] += a * s
        mag[t, e] += m * s
        if not renormalize and scoring == "softmax":
            p = torch.softmax(row, 0)
            dl[t] -= p * (g * d).sum()
            mag[t] += p * (g * d).abs().sum()
    return gates, experts, dl, mag


def _run(logits, k, dgates=None, **kw):
    from mace_onegpu.experts import route
    x = logits.cuda()
    bias = kw.pop("bias", None)
    kw["bias"] = bias.cuda() if bias is not None else None
    if dgates is None:
        gates, experts = route(x, k, **kw)
        return gates.cpu().double(), experts.cpu(), None
    x = x.requires_grad_()
    gates, experts = route(x, k, **kw)
    (dl,) = torch.autograd.grad(gates, x, dgates.cuda())
    assert dl.dtype == logits.dtype
    return gates.detach().cpu().double(), experts.cpu(), dl.cpu().double()


def _check(logits, k, dgates=None, **kw):
    full = dict(dict(scoring="softmax", bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0), **kw)
    gates, experts, dl, mag = _reference(logits, k, dgates=dgates, **full)
    g, e, d = _run(logits, k, dgates, **full)
    assert torch.equal(e, experts)
    assert bool(((g - gates).abs() <= 96 * U * gates.abs() + 1e-37).all()), float((g - gates).abs().max())
    if dgates is not None:
        tiny = 2.0 ** -25 if logits.dtype == torch.float16 else 1e-37
        bound = 256 * U * mag + HALF_ULP[logits.dtype] * dl.abs() + tiny
        assert bool(((d - dl).abs() <= bound).all()), float(((d - dl).abs() - bound).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (67, 5, 5), (130, 16, 2), (65, 17, 3), (33, 64, 6),
                                   (70, 89, 3), (20, 128, 8), (40, 256, 8), (9, 300, 32), (5, 1024, 17)])
def test_choice_gates_and_gradient(T, E, k, renormalize, scoring, dtype):
    g = torch.Generator().manual_seed(1000 * T + E + k)
    logits = (1.5 * torch.randn(T, E, generator=g)).to(dtype)
    bias = 0.5 * torch.randn(E, generator=g)
    dgates = torch.randn(T, k, generator=g)
    _check(logits, k, dgates, scoring=scoring, renormalize=renormalize, bias=bias, scale=2.5)
    _check(logits, k, scoring=scoring, renormalize=renormalize)


@pytest.mark.parametrize("E,groups,top_groups,k", [(8, 2, 1, 2), (64, 8, 3, 6), (256, 8, 4, 8), (60, 5, 2, 4),
                                                   (64, 64, 5, 5), (256, 64, 40, 9), (39, 3, 1, 20), (512, 8, 8, 8)])
def test_groups(E, groups, top_groups, k):
    g = torch.Generator().manual_seed(E + groups)
    logits = torch.randn(45, E, generator=g)
    logits[:, ::3] = -math.inf                     # some groups of few or no open experts
    logits[3] = -math.inf
    bias = 0.5 * torch.randn(E, generator=g)
    for kw in (dict(scoring="sigmoid", bias=bias), dict(renormalize=False)):
        _check(logits, k, torch.randn(45, k, generator=g), groups=groups, top_groups=top_groups, **kw)


@pytest.mark.parametrize("E,k", [(7, 3), (64, 8), (200, 16), (1000, 9)])
def test_ties_go_to_the_lowest_index(E, k):
    g = torch.Generator().manual_seed(E)
    logits = torch.randint(-2, 3, (51, E), generator=g).to(torch.bfloat16)
    logits[0] = 0
    logits[1] = torch.where(torch.arange(E) % 2 == 0, 0.0, -0.0)     # -0 and 0 are equal
    _check(logits, k)
    _check(logits, k, bias=torch.randint(-1, 2, (E,), generator=g).float())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_closed_experts_and_extreme_logits(renormalize, scoring):
    g = torch.Generator().manual_seed(4)
    E, k, T = 24, 4, 12
    logits = torch.randn(T, E, generator=g)
    logits[0] = -math.inf                                            # nothing open
    logits[1, 2:] = -math.inf                                        # fewer open than k
    logits[2] = torch.finfo(torch.float32).min                       # the lowest value is a value
    logits[3, 5:] = torch.finfo(torch.float32).min
    logits[4] = -200 + 20 * torch.rand(E, generator=g)               # every sigmoid and many exponentials underflow
    logits[5] = 200 + 20 * torch.rand(E, generator=g)                # every sigmoid is 1
    logits[6, 1:] = -math.inf
    logits[7] = 1e30
    logits[7, 3] = -1e30
    dgates = torch.randn(T, k, generator=g)
    dgates[0] = math.nan                                             # of slots that hold nothing
    _check(logits, k, dgates, scoring=scoring, renormalize=renormalize)
    closing = torch.zeros(E)
    closing[3] = -math.inf                                           # a bias may close an expert as well
    _check(logits[1:], k, dgates[1:], scoring=scoring, renormalize=renormalize, bias=closing)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_not_a_number_is_not_hidden(scoring):
    logits = torch.randn(5, 30, generator=torch.Generator().manual_seed(1))
    logits[2, 7] = math.nan
    g, e, _ = _run(logits, 3, scoring=scoring)
    assert e[2, 0] == 7 and g[2].isnan().all()
    others = [0, 1, 3, 4]
    g0, e0, _ = _run(logits[others], 3, scoring=scoring)
    assert torch.equal(e[others], e0) and torch.equal(g[others], g0)
    assert ((e >= 0) & (e < 30)).all()


def test_strided_logits_many_rows_and_no_rows():
    from mace_onegpu.experts import route
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(30011, 40, generator=g).cuda()
    for view in (wide[:, 3:36], wide[::2, :16], wide[:, ::2], wide.t()[:, :20], wide[:1].expand(9, 40)):
        for a, b in zip(route(view, 4), route(view.contiguous(), 4)):
            assert torch.equal(a, b)
    gates, experts = route(wide, 5)
    top = torch.sort(wide, dim=1, descending=True, stable=True)
    assert torch.equal(experts.long(), top.indices[:, :5])
    assert torch.allclose(gates, torch.softmax(top.values[:, :5], 1), rtol=96 * U, atol=0)
    x = torch.empty(0, 40, device="cuda", requires_grad=True)
    gates, experts = route(x, 5)
    (dx,) = torch.autograd.grad(gates, x, torch.empty(0, 5, device="cuda"))
    assert gates.shape == experts.shape == (0, 5) and dx.shape == (0, 40)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_against_differences(renormalize, scoring):
    """Logits far enough apart that no choice changes within the step: <grad, v> against central differences."""
    from mace_onegpu.experts import route
    g = torch.Generator().manual_seed(6)
    T, E, k, h = 50, 20, 3, 5e-3
    logits = torch.stack([torch.randperm(E, generator=g) * 0.3 for _ in range(T)]).cuda().requires_grad_()
    dg, v = torch.randn(T, k, generator=g).cuda(), torch.randn(T, E, generator=g).cuda()
    kw = dict(scoring=scoring, renormalize=renormalize)
    (dl,) = torch.autograd.grad(route(logits, k, **kw)[0], logits, dg)
    with torch.no_grad():
        f = [float((route(logits + s * h * v, k, **kw)[0].double() * dg).sum()) for s in (1, -1)]
    want = float((dl.double() * v).sum())
    assert abs((f[0] - f[1]) / (2 * h) - want) < 1e-3 * float((dl * v).abs().sum())


def test_graph_replay():
    from mace_onegpu.experts import plan_experts, route
    g = torch.Generator().manual_seed(3)
    x = torch.randn(700, 16, generator=g).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gates, experts = route(x, 2)
        plan = plan_experts(experts, 16)
    for _ in range(3):
        x.copy_(torch.randn(700, 16, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        g0, e0 = route(x, 2)
        p0 = plan_experts(e0, 16)
        assert torch.equal(gates, g0) and torch.equal(experts, e0)
        assert torch.equal(plan.offsets, p0.offsets) and torch.equal(plan.order, p0.order)
