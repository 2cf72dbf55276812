"""linear_cross_entropy and its gradients against the formula in 64 bits on the same (rounded) inputs.

Tolerances, element by element, u = 2^-24, P products for one (6 of float32's parts, else 1): a sum of n products has at
most P n roundings on any path, and the parts left out of a float32 product are below 3 u of it.  So a logit is off by
(P D + 4) u sum|x w|; an exponential of z adds (4 + |z|) u of its value; d is rounded to the type (half a unit in its
last place; float16, scaled by 2^14: to 2^-39 at least).  The sums of exponentials have at most 64 + classes / 64
roundings.  Rounding to the output's type adds half a unit of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(T, D, V, dtype, seed, ignored=0.2):
    g = torch.Generator().manual_seed(seed)
    w = 2 / D ** 0.5 * torch.randn(V, D, generator=g)
    y = torch.randint(0, V, (T,), generator=g)
    x = (torch.randn(T, D, generator=g) + 3 * torch.rand(T, 1, generator=g) * w[y]).to(dtype)
    y[torch.rand(T, generator=g) < ignored] = -100
    return x, w.to(dtype), y, 0.1 + torch.rand(T, generator=g)


def _reference(x, w, y, dloss, reduction, dtype):
    x, w = x.double(), w.double()
    (T, D), V = x.shape, w.shape[0]
    P = 6 if dtype == torch.float32 else 1
    asked = y >= 0
    at = y.clamp_min(0)
    logits = x @ w.T.contiguous()
    el = (P * D + 4) * U * (x.abs() @ w.abs().T.contiguous())
    lse = torch.logsumexp(logits, 1)
    picked = logits.gather(1, at[:, None]).squeeze(1)
    depth = logits.amax(1, keepdim=True) - logits
    p = torch.exp(logits - lse[:, None])
    elz = (p * (el + U * (8 + depth))).sum(1) + U * (64 + V / 64 + 2 * lse.abs())
    loss = torch.where(asked, lse - picked, 0.0)
    eloss = torch.where(asked, elz + el.gather(1, at[:, None]).squeeze(1) + 2 * U * (lse.abs() + picked.abs()), 0.0)
    n = max(1, int(asked.sum()))
    if reduction == "none":
        g, out, eout = dloss.double(), loss, eloss
    else:
        f = 1 / n if reduction == "mean" else 1.0
        g = torch.full((T,), f, dtype=torch.float64, device=x.device)
        out, eout = loss.sum() * f, eloss.sum() * f + 64 * U * loss.abs().sum() * f
    g = torch.where(asked, g, 0.0)[:, None]
    d = p.scatter_add(1, at[:, None], torch.full((T, 1), -1.0, dtype=torch.float64, device=x.device))
    ed = (p * (el + elz[:, None] + U * (8 + (logits - lse[:, None]).abs())) + 8 * U * d.abs()
          + (4 * U if dtype == torch.float32 else HALF_ULP[dtype]) * d.abs() + 2.0 ** -39 * (dtype == torch.float16))
    ad, aw, ax, ag = d.abs(), w.abs(), x.abs(), g.abs()
    dx, dw = (g * d) @ w, (g * d).T.contiguous() @ x
    edx = ag * ((ed + (P * V + 8) * U * ad) @ aw)
    # float16: a row's weight enters the rounded d as its share of the largest
    edw = (ag * (ed + (P * T + 16) * U * ad)).T.contiguous() @ ax
    if dtype == torch.float16:
        edw += float(ag.max()) * 2.0 ** -39 * ax.sum(0, keepdim=True)
    ref = dict(loss=out, dx=dx, dw=dw)
    bound = dict(loss=eout + U * out.abs() + 1e-37, dx=edx + HALF_ULP[dtype] * dx.abs() + TINY[dtype],
                 dw=edw + HALF_ULP[dtype] * dw.abs() + TINY[dtype])
    return ref, bound


def _check(got, ref, bound):
    for name, t in got.items():
        err = (t.detach().double().reshape(ref[name].shape) - ref[name].to(t.device)).abs()
        assert bool((err <= bound[name].to(t.device)).all()), (name, float((err - bound[name].to(t.device)).max()))


def _run(x, w, y, dloss, reduction, **kw):
    from mace_onegpu.cross_entropy import linear_cross_entropy
    x, w = (t.detach().cuda().clone().requires_grad_() for t in (x, w))
    loss = linear_cross_entropy(x, w, y.cuda(), reduction=reduction, **kw)
    assert loss.dtype == torch.float32 and loss.shape == (y.shape if reduction == "none" else ())
    up = dloss.cuda() if reduction == "none" else torch.ones((), device="cuda")
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, y.cuda(), reduction=reduction, **kw), loss)
    return dict(loss=loss, dx=dx, dw=dw)


SIZES = [(1, 1, 1), (1, 128, 89), (2, 3, 2), (17, 24, 19), (64, 64, 64), (130, 200, 300), (129, 128, 128),
         (300, 65, 1000), (1000, 32, 130), (5, 777, 2003), (257, 1000, 515), (2000, 16, 7), (9, 40, 70001),
         (3, 2500, 33), (513, 256, 769), (2047, 200, 6201), (2048, 2112, 6144)]


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,V", SIZES)
def test_loss_and_gradients(T, D, V, dtype, reduction):
    if T * V * D > 1e9 and reduction != "none":
        pytest.skip("large tiles: once a type")
    x, w, y, dloss = (t.cuda() for t in _inputs(T, D, V, dtype, T + D + V))
    ref, bound = _reference(x, w, y, dloss, reduction, dtype)
    _check(_run(x, w, y, dloss, reduction), ref, bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_several_pieces_of_the_classes(dtype):
    x, w, y, dloss = (t.cuda() for t in _inputs(40000, 24, 5000, dtype, 1))
    ref, bound = _reference(x, w, y, dloss, "none", dtype)
    got = _run(x, w, y, dloss, "none")
    _check(got, ref, bound)
    again = _run(x, w, y, dloss, "none")
    assert all(torch.equal(got[n], again[n]) for n in got)       # no order of sums changes from run to run


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_left_out(dtype):
    """None, most and all rows ignored, also where they hold infinities and NaN, by an index of the caller's."""
    x, w, y, dloss = _inputs(200, 48, 90, dtype, 3, ignored=0.0)
    for share in (0.0, 0.9, 1.0):
        out = torch.rand(200, generator=torch.Generator().manual_seed(4)) < share
        z = y.masked_fill(out, 7777)
        dirty = x.clone()
        dirty[out] = float("nan")
        dirty[out, ::2] = float("inf")
        weights = dloss.masked_fill(out, float("nan"))
        for reduction in ("mean", "none"):
            ref, bound = _reference(x.cuda(), w.cuda(), y.masked_fill(out, -1).cuda(), dloss.cuda(), reduction, dtype)
            got = _run(dirty, w, z, weights, reduction, ignore_index=7777)
            _check(got, ref, bound)
            assert not got["dx"][out.cuda()].any()
            if share == 1.0:
                assert not got["loss"].any() and not got["dw"].any()


def test_only_one_gradient():
    from mace_onegpu.cross_entropy import linear_cross_entropy
    x, w, y, _ = (t.cuda() for t in _inputs(70, 48, 90, torch.float32, 5))
    both = _run(x, w, y, y, "mean")
    for i, name in enumerate(("dx", "dw")):
        args = [t.clone().requires_grad_(q == i) for q, t in enumerate((x, w))]
        (d,) = torch.autograd.grad(linear_cross_entropy(*args, y), args[i])
        assert torch.equal(d, both[name])


def test_shapes_strides_and_target_types():
    from mace_onegpu.cross_entropy import linear_cross_entropy as f
    x, w, y, _ = (t.cuda() for t in _inputs(60, 48, 90, torch.bfloat16, 6))
    want = f(x, w, y, reduction="none")
    assert torch.equal(f(x.view(3, 20, 48), w, y.view(3, 20), reduction="none"), want.view(3, 20))
    assert torch.equal(f(x, w, y.int(), reduction="none"), want)
    wide = torch.zeros(60, 3, 50, dtype=torch.bfloat16, device="cuda")
    wide[:, 1, 1:49] = x
    assert torch.equal(f(wide[:, 1, 1:49], w, y, reduction="none"), want)
    off = torch.zeros(90 * 48 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(90, 48)
    off.copy_(w)
    assert torch.equal(f(x, off, y, reduction="none"), want)
    assert torch.equal(f(x, w.t().contiguous().t(), y, reduction="none"), want)
    assert torch.equal(f(x[7], w, y[7], reduction="none"), f(x[7:8], w, y[7:8], reduction="none")[0])
    assert torch.equal(f(x, w, torch.stack([y, y], 1)[:, 0], reduction="none"), want)
    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(f(xg, w, y, reduction="none").sum(), xg)          # an expanded cotangent
    (dx1,) = torch.autograd.grad(f(xg, w, y, reduction="sum"), xg)
    assert torch.equal(dx, dx1)


def test_no_rows():
    from mace_onegpu.cross_entropy import linear_cross_entropy as f
    w = torch.randn(9, 8, device="cuda", requires_grad=True)
    x = torch.empty(0, 8, device="cuda", requires_grad=True)
    y = torch.empty(0, dtype=torch.long, device="cuda")
    for reduction in ("mean", "sum", "none"):
        loss = f(x, w, y, reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
        assert not loss.any() and dx.shape == (0, 8) and not dw.any() and dw.shape == (9, 8)


def test_far_logits_and_bad_targets_and_non_finite_rows():
    from mace_onegpu.cross_entropy import linear_cross_entropy as f
    x = torch.tensor([[300.0, 0], [0, 300.0], [-300.0, 300.0], [1, 2], [3, 4], [float("nan"), 0], [float("inf"), 1]])
    w, y = torch.tensor([[10.0, 0], [0, 10.0], [0, 0]]), torch.tensor([0, 0, 1, 3, -1, 0, 1])
    loss = f(x.cuda(), w.cuda(), y.cuda(), reduction="none").cpu()
    assert loss[:3].tolist() == [0.0, 3000.0, 0.0] and loss[3:].isnan().all()
    xg, wg = x[:5].cuda().requires_grad_(), w.cuda().requires_grad_()
    dx, dw = torch.autograd.grad(f(xg, wg, y[:5].cuda(), reduction="sum"), (xg, wg))
    assert dx[3:].isnan().all() and dw.isnan().all()
    assert dx[:3].tolist() == [[0.0, 0.0], [-10.0, 10.0], [0.0, 0.0]]


def test_weights_of_very_different_size():
    """A row's weight of 2^-40 of the largest keeps its own dx."""
    for dtype in DTYPES:
        x, w, y, _ = (t.cuda() for t in _inputs(50, 32, 40, dtype, 8, ignored=0.0))
        dloss = torch.ones(50, device="cuda")
        dloss[::2] = 2.0 ** -10 if dtype == torch.float16 else 2.0 ** -40
        ref, bound = _reference(x, w, y, dloss, "none", dtype)
        _check(_run(x, w, y, dloss, "none"), ref, bound)
    x, w, y, _ = (t.cuda() for t in _inputs(50, 32, 40, torch.float32, 8, ignored=0.0))
    got = _run(x, w, y, torch.zeros(50), "none")
    assert not got["dx"].any() and not got["dw"].any()


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_gradient_against_differences(reduction):
    from mace_onegpu.cross_entropy import linear_cross_entropy
    x, w, y, dloss = (t.cuda() for t in _inputs(33, 40, 50, torch.float32, 9))
    up = dloss if reduction == "none" else torch.ones((), device="cuda")
    args = [x.requires_grad_(), w.requires_grad_()]
    f = lambda a: linear_cross_entropy(a[0], a[1], y, reduction=reduction)  # noqa: E731
    grads = torch.autograd.grad(f(args), args, up)
    g, h = torch.Generator().manual_seed(1), 1e-2
    for i in range(2):
        v = torch.randn(args[i].shape, generator=g).cuda()
        with torch.no_grad():
            s = [float((f([a + sign * h * v if q == i else a for q, a in enumerate(args)]).double() * up).sum())
                 for sign in (1, -1)]
        slope, want = (s[0] - s[1]) / (2 * h), float((grads[i].double() * v.double()).sum())
        assert abs(slope - want) < 2e-3 * float((grads[i].double() * v.double()).abs().sum()), (i, slope, want)


def test_another_stream_and_graph_replay():
    """A captured forward and backward whose rows, weights and targets (how many are ignored too) change."""
    from mace_onegpu.cross_entropy import linear_cross_entropy
    x, w, y, _ = (t.cuda() for t in _inputs(300, 64, 200, torch.bfloat16, 10))
    want = linear_cross_entropy(x, w, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear_cross_entropy(x, w, y)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    xs, ws, ys = x.clone().requires_grad_(), w.clone().requires_grad_(), y.clone()

    def step():
        loss = linear_cross_entropy(xs, ws, ys)
        return (loss.detach(), *torch.autograd.grad(loss, (xs, ws)))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed, ignored in ((11, 0.0), (12, 0.95), (13, 1.0), (14, 0.3)):
        a, b, c, _ = _inputs(300, 64, 200, torch.bfloat16, seed, ignored)
        with torch.no_grad():
            xs.copy_(a)
            ws.copy_(b)
        ys.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))


def test_refusals():
    from mace_onegpu.cross_entropy import linear_cross_entropy as f
    x, w, y, _ = (t.cuda() for t in _inputs(10, 8, 6, torch.float32, 12))
    for error, call in [(TypeError, lambda: f(x.cpu(), w, y)), (TypeError, lambda: f(x, w.cpu(), y)),
                        (TypeError, lambda: f(x, w, y.cpu())), (TypeError, lambda: f(x, w.half(), y)),
                        (TypeError, lambda: f(x.double(), w.double(), y)), (TypeError, lambda: f(x, w, y.float())),
                        (ValueError, lambda: f(x, w[:, :7], y)), (ValueError, lambda: f(x, w[:0], y)),
                        (ValueError, lambda: f(x, w[None], y)), (ValueError, lambda: f(x, w, y[:9])),
                        (ValueError, lambda: f(x[:, :0], w[:, :0], y)),
                        (ValueError, lambda: f(x, w, y, reduction="max"))]:
        with pytest.raises(error):
            call()
    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(f(xg, w, y), xg, create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        dx.sum().backward()


@pytest.mark.parametrize("T,V", [(1, 50), (5, 700), (16, 33), (17, 50), (130, 700), (600, 5000)])
def test_probabilities_sum_to_one(T, V):
    """sum_v dW[v] = g x sum_v d, and d of a row sums to 0 whatever the logits' roundings, if both directions take the
    same logits: here near 2000, where a rounded log of the sum alone would be off by up to 2^-14.  One asked row, as
    sums over rows have no roundings then.  E[depth] <= log V; sum |d| <= 2."""
    from mace_onegpu.cross_entropy import linear_cross_entropy
    g = torch.Generator().manual_seed(T + V)
    base = torch.randn(33, generator=g)
    w = base + 0.02 * torch.randn(V, 33, generator=g)
    x = (2000 / base.square().sum() * base).expand(T, 33).contiguous()
    y = torch.full((T,), -100)
    y[T // 2] = V // 3
    wg = w.cuda().requires_grad_()
    loss = linear_cross_entropy(x.cuda(), wg, y.cuda(), reduction="sum")
    dw, = torch.autograd.grad(loss, wg)
    bound = U * x[0].double().abs() * (16 + 2 * torch.tensor(float(V)).log() + 64 + V / 64 + 2 * (6 + 16))
    assert float(dw.abs().max()) > 0.01
    assert bool((dw.double().sum(0).cpu().abs() <= bound).all()), float((dw.double().sum(0).cpu().abs() / bound).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,V", [(1, 16, 8), (16, 1000, 3), (9, 77, 3000), (3, 5000, 65), (16, 40, 70001)])
def test_few_rows_with_gradients(T, D, V, dtype):
    x, w, y, dloss = _inputs(T, D, V, dtype, T + D + V)
    for reduction in ("mean", "none"):
        ref, bound = _reference(x.cuda(), w.cuda(), y.cuda(), dloss.cuda(), reduction, dtype)
        _check(_run(x, w, y, dloss, reduction), ref, bound)


@pytest.mark.parametrize("T,D,V,dtype", [(16, 64, 200, torch.float32), (1, 128, 20000, torch.bfloat16),
                                         (3, 777, 5000, torch.float16), (200, 32, 20000, torch.bfloat16)])
def test_few_rows_in_a_replayed_graph(T, D, V, dtype):
    """Few rows of many classes; ignored rows hold NaN, and how many there are changes between the replays."""
    from mace_onegpu.cross_entropy import linear_cross_entropy
    x, w, y, dloss = (t.cuda() for t in _inputs(T, D, V, dtype, 10))
    xs, ws, ys, up = x.clone().requires_grad_(), w.clone().requires_grad_(), y.clone(), dloss.clone()

    def step():
        loss = linear_cross_entropy(xs, ws, ys, reduction="none")
        return (loss.detach(), *torch.autograd.grad(loss, (xs, ws), up))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed, ignored in ((11, 0.0), (12, 0.5), (13, 1.0), (14, 0.3)):
        a, b, c, d = (t.cuda() for t in _inputs(T, D, V, dtype, seed, ignored))
        a[c < 0] = float("nan")
        with torch.no_grad():
            xs.copy_(a)
            ws.copy_(b)
        ys.copy_(c)
        up.copy_(d)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(p, q) and bool(q.isfinite().all()) for p, q in zip(out, want))
        assert not bool(out[1][c < 0].any())


@pytest.mark.parametrize("T", [16384, 16385, 70001, 4194304 + 5000])
def test_lists_of_many_rows(T):
    """Every row's loss and gradient, where the asked rows are listed by one workgroup, by many, by larger ones."""
    from mace_onegpu.cross_entropy import linear_cross_entropy
    x, w, y, dloss = (t.cuda() for t in _inputs(T, 4, 5, torch.float32, T, 0.7))
    ref, bound = _reference(x, w, y, dloss, "none", torch.float32)
    got = linear_cross_entropy(x, w, y.int(), reduction="none")
    xs = x.requires_grad_()
    dx, = torch.autograd.grad(linear_cross_entropy(xs, w, y, reduction="none"), xs, dloss)
    _check(dict(loss=got, dx=dx), ref, bound)
