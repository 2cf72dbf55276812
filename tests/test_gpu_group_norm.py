"""group_norm and its gradients against the formula in 64 bits on the same (rounded) inputs.

Tolerances, element by element, u = 2^-24: a sum of n values by threads, lanes, waves, channels and tiles has fewer than
CHAIN = 160 roundings on any path (16 rows of a thread, 6 lane moves, 16 sets, 64 channels a lane, 20 tiles a thread and
the moves between them), so a mean is off by at most CHAIN u mean|x|, a variance and a sum of products by CHAIN u of
theirs.  The activations add 16 u of their terms (their slopes are at most 1.13, their second derivatives at most 0.8),
other operations less than 8 u.  Rounding to the output's type adds half a unit in its last place."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
CHAIN = 160
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(rows, C, dtype, p_dtype, seed, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, C, generator=g) * torch.exp(0.5 * torch.randn(rows, 1, generator=g)) + offset).to(dtype)
    w = (1 + 0.2 * torch.randn(C, generator=g)).to(p_dtype)
    b = (0.2 * torch.randn(C, generator=g)).to(p_dtype)
    return x, w, b, torch.randn(rows, C, generator=g).to(dtype)


def _act(z, kind):
    if kind == "silu":
        q = torch.sigmoid(z)
        return z * q, q * (1 + z * (1 - q))
    if kind == "gelu":
        q = torch.special.ndtr(z)
        return z * q, q + z * torch.exp(-z * z / 2) * 0.3989422804014327
    return z, torch.ones_like(z)


def _reference(x, w, b, dy, bounds, G, eps, kind, dtype, p_dtype):
    """Results and bounds of their errors; bounds: first row of every structure and the end of the last."""
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    C = x.shape[1]
    out = {n: torch.zeros_like(x) for n in ("y", "dx", "ey", "edx")}
    sums = {n: torch.zeros(C, dtype=torch.float64) for n in ("dw", "db", "edw", "edb", "adw", "adb")}
    for r0, r1 in zip(bounds[:-1], bounds[1:]):
        if r1 <= r0:
            continue
        v, d = x[r0:r1].view(r1 - r0, G, -1), dy[r0:r1].view(r1 - r0, G, -1)
        wg, bg = w.view(G, -1), b.view(G, -1)
        mean = lambda t: t.mean((0, 2), keepdim=True)  # noqa: E731
        mu = mean(v)
        r = 1 / torch.sqrt(mean((v - mu) ** 2) + eps)
        h = (v - mu) * r
        z = h * wg + bg
        y, slope = _act(z, kind)
        dz = d * slope
        g = dz * wg
        m0, m1 = mean(g), mean(g * h)
        dx = r * (g - m0 - h * m1)
        eh = U * (r * (CHAIN * mean(v.abs()) + 8 * v.abs()) + CHAIN * h.abs())
        ez = eh * wg.abs() + 8 * U * ((h * wg).abs() + bg.abs())
        ey = 1.13 * ez + 16 * U * (z.abs() + y.abs())
        edz = d.abs() * (0.8 * ez * (kind != "none") + 16 * U * (1 + z.abs()))
        eg = wg.abs() * edz + 2 * U * g.abs()
        em0 = mean(eg) + CHAIN * U * mean(g.abs())
        em1 = mean(eg * h.abs() + g.abs() * eh) + CHAIN * U * mean((g * h).abs())
        edx = r * (eg + em0 + h.abs() * em1 + eh * m1.abs() + CHAIN * U * (g.abs() + m0.abs() + (h * m1).abs()))
        for name, t in (("y", y), ("dx", dx), ("ey", ey), ("edx", edx)):
            out[name][r0:r1] = t.reshape(r1 - r0, C)
        flat = lambda t: t.sum(0).reshape(C)  # noqa: E731
        sums["dw"] += flat(dz * h)
        sums["db"] += flat(dz)
        sums["edw"] += flat(edz * h.abs() + dz.abs() * eh)
        sums["edb"] += flat(edz)
        sums["adw"] += flat((dz * h).abs())
        sums["adb"] += flat(dz.abs())
    chain = 2 * CHAIN + x.shape[0] / 1024       # a thread's rows over all its structures
    ref = dict(y=out["y"], dx=out["dx"], dw=sums["dw"], db=sums["db"])
    tiny = {t: 2.0 ** -25 if t == torch.float16 else 1e-37 for t in DTYPES}
    bound = dict(y=out["ey"] + HALF_ULP[dtype] * out["y"].abs() + tiny[dtype],
                 dx=out["edx"] + HALF_ULP[dtype] * out["dx"].abs() + tiny[dtype],
                 dw=sums["edw"] + chain * U * sums["adw"] + HALF_ULP[p_dtype] * sums["dw"].abs() + tiny[p_dtype],
                 db=sums["edb"] + chain * U * sums["adb"] + HALF_ULP[p_dtype] * sums["db"].abs() + tiny[p_dtype])
    return ref, bound


def _check(got, ref, bound):
    for name, t in got.items():
        err = (t.detach().double().cpu().reshape(ref[name].shape) - ref[name]).abs()
        assert bool((err <= bound[name]).all()), (name, float((err - bound[name]).max()))


def _run(x, w, b, dy, G, kind, offsets=None, eps=1e-5):
    from mace_onegpu.group_norm import group_norm
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    act = None if kind == "none" else kind
    y = group_norm(leaves[0], G, leaves[1], leaves[2], eps, act, offsets)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    with torch.no_grad():
        assert torch.equal(group_norm(*leaves[:1], G, *leaves[1:], eps, act, offsets), y)
    return dict(zip(("y", "dx", "dw", "db"), (y, *grads)))


UNIFORM = [(1, 1, 1, 1), (3, 1, 8, 8), (5, 17, 24, 3), (2, 200, 128, 8), (1, 1000, 96, 4), (7, 33, 40, 5),
           (4, 3, 130, 10), (2, 70, 2048, 1), (1, 9, 4096, 1), (3, 5, 30, 30), (1, 5000, 16, 1), (2, 300, 1030, 2),
           (300, 2, 6, 2), (1500, 3, 64, 2), (1, 257, 1, 1), (1, 70001, 8, 2)]


@pytest.mark.parametrize("kind", ["none", "silu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("structs,each,C,G", UNIFORM)
def test_structures_of_equal_size(structs, each, C, G, dtype, kind):
    x, w, b, dy = _inputs(structs * each, C, dtype, dtype, structs + each + C)
    ref, bound = _reference(x, w, b, dy, [each * s for s in range(structs + 1)], G, 1e-5, kind, dtype, dtype)
    got = _run(x.view(structs, each, C), w, b, dy.view(structs, each, C), G, kind)
    assert got["y"].shape == (structs, each, C) and got["y"].dtype == dtype
    _check(got, ref, bound)


RAGGED = [[0, 1], [0, 0, 0, 3, 3, 10], [5, 9, 9, 40, 41, 60], [0, 3000], [0, 700, 701, 1500, 1500, 4000],
          [17, 18, 900, 2500, 2501, 2502, 2502], list(range(0, 400, 3)), [3, 3], [0, 256, 512, 769, 1024, 1281]]


@pytest.mark.parametrize("dtype,p_dtype", [(t, t) for t in DTYPES] + [(torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("C,G", [(128, 8), (24, 3), (70, 2), (5, 1)])
@pytest.mark.parametrize("at", range(len(RAGGED)))
def test_ragged_structures(at, C, G, dtype, p_dtype):
    bounds = RAGGED[at]
    rows = bounds[-1] + (at % 3) * 11
    x, w, b, dy = _inputs(rows, C, dtype, p_dtype, at + C)
    ref, bound = _reference(x, w, b, dy, bounds, G, 1e-5, "silu", dtype, p_dtype)
    got = _run(x, w, b, dy, G, "silu", torch.tensor(bounds, dtype=torch.int32).cuda())
    _check(got, ref, bound)
    outside = torch.ones(rows, dtype=torch.bool)
    outside[bounds[0]:bounds[-1]] = False
    assert not got["y"][outside.cuda()].any() and not got["dx"][outside.cuda()].any()
    long = _run(x, w, b, dy, G, "silu", torch.tensor(bounds).cuda())
    assert all(torch.equal(got[n], long[n]) for n in got)


def test_ragged_equals_uniform():
    from mace_onegpu.group_norm import group_norm
    x = torch.randn(6, 50, 96, generator=torch.Generator().manual_seed(0)).cuda()
    o = torch.arange(0, 301, 50, device="cuda")
    assert float((group_norm(x, 4, activation="gelu").view(300, 96)
                  - group_norm(x.view(300, 96), 4, activation="gelu", offsets=o)).abs().max()) < 64 * U * 8


def test_strides_and_absent_parameters_and_module():
    from mace_onegpu.group_norm import GroupNorm, group_norm
    g = torch.Generator().manual_seed(1)
    feats = torch.randn(3, 33, 4, 128, generator=g).cuda()
    w, b = torch.randn(128, generator=g).cuda(), torch.randn(128, generator=g).cuda()
    x = feats[:, :, 0]
    want = group_norm(x.contiguous(), 8, w, b, activation="silu")
    assert torch.equal(group_norm(x, 8, w, b, activation="silu"), want)
    assert torch.equal(group_norm(x.transpose(1, 2).contiguous().transpose(1, 2), 8, w, b, activation="silu"), want)
    assert torch.equal(group_norm(feats[::2, ::3, 1, 1:100], 9), group_norm(feats[::2, ::3, 1, 1:100].contiguous(), 9))
    assert torch.equal(group_norm(x.unflatten(1, (3, 11)), 8, w, b, activation="silu").flatten(1, 2), want)
    one, zero = torch.ones(128, device="cuda"), torch.zeros(128, device="cuda")
    assert torch.equal(group_norm(x, 8), group_norm(x, 8, one, zero))
    assert torch.equal(group_norm(x, 8, None, b), group_norm(x, 8, one, b))
    m = GroupNorm(8, 128, activation="gelu", device="cuda")
    assert torch.equal(m(x), group_norm(x, 8, activation="gelu"))
    xg = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(m(xg).sum(), xg)                    # an expanded cotangent
    (dx1,) = torch.autograd.grad(m(xg), xg, torch.ones(3, 33, 128, device="cuda"))
    assert torch.equal(dx, dx1)
    m(x).square().sum().backward()
    assert m.weight.grad.shape == (128,) and m.bias.grad.shape == (128,)


def test_no_rows_and_constant_and_non_finite_structures():
    from mace_onegpu.group_norm import group_norm
    w = torch.ones(40, device="cuda", requires_grad=True)
    b = torch.ones(40, device="cuda", requires_grad=True)
    for x, o in ((torch.empty(0, 7, 40), None), (torch.empty(4, 0, 40), None), (torch.empty(0, 40), [0, 0, 0])):
        x = x.cuda().requires_grad_()
        y = group_norm(x, 4, w, b, offsets=None if o is None else torch.tensor(o).cuda())
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(x))
        assert y.shape == dx.shape == x.shape and not dw.any() and not db.any()
    x = torch.full((3, 5, 40), 7.0, device="cuda")
    x[1, 2, 5], x[2, 4, 39] = float("nan"), float("inf")
    with torch.no_grad():
        y = group_norm(x, 4, w, b)
    bad = torch.zeros(3, 5, 4, 10, dtype=torch.bool, device="cuda")
    bad[1, :, 0], bad[2, :, 3] = True, True
    bad = bad.view(3, 5, 40)
    assert torch.equal(y[~bad], torch.ones_like(y[~bad])) and y[bad].isnan().all()
    # what stands in rows outside the structures does not matter, forward or backward
    x = torch.randn(60, 40, generator=torch.Generator().manual_seed(2)).cuda()
    o = torch.tensor([5, 20, 50]).cuda()
    dirty = x.clone()
    dirty[:5], dirty[50:] = float("nan"), float("inf")
    got = [_run(t.cpu(), w.detach().cpu(), b.detach().cpu(), t.cpu(), 4, "silu", o) for t in (x, dirty)]
    assert all(torch.equal(got[0][n], got[1][n]) for n in got[0])


def test_offsets_out_of_range_stay_inside():
    """Ends past the rows there are and negative ones are cut: the kernels touch nothing outside."""
    from mace_onegpu.group_norm import group_norm
    whole = torch.randn(100, 32, generator=torch.Generator().manual_seed(3)).cuda()
    y = group_norm(whole[:40], 4, offsets=torch.tensor([-7, 10, 1000], device="cuda"))
    assert torch.equal(y, group_norm(whole[:40], 4, offsets=torch.tensor([0, 10, 40], device="cuda")))
    y = group_norm(whole[:40], 4, offsets=torch.tensor([-7, 10, 2 ** 40], device="cuda"))
    assert torch.equal(y, group_norm(whole[:40], 4, offsets=torch.tensor([0, 10, 40], device="cuda")))


@pytest.mark.parametrize("offsets", [None, [0, 3, 3, 22]])
@pytest.mark.parametrize("kind", ["none", "silu", "gelu"])
def test_gradient_against_differences(kind, offsets):
    """<grad, v> against (f(x + h v) - f(x - h v)) / 2 h, f summed in 64 bits: off by O(h^2) and roundings of f over
    h."""
    from mace_onegpu.group_norm import group_norm
    x, w, b, dy = (t.cuda() for t in _inputs(22, 48, torch.float32, torch.float32, 5))
    o = None if offsets is None else torch.tensor(offsets).cuda()
    shape = (2, 11, 48) if o is None else (22, 48)
    g = torch.Generator().manual_seed(9)
    args = [t.requires_grad_() for t in (x.view(shape), w, b)]
    f = lambda a: group_norm(a[0], 4, a[1], a[2], activation=None if kind == "none" else kind, offsets=o)  # noqa: E731
    grads = torch.autograd.grad(f(args), args, dy.view(shape))
    h = 1e-2
    for i in range(3):
        v = torch.randn(args[i].shape, generator=g).cuda()
        with torch.no_grad():
            s = [float((f([a + sign * h * v if q == i else a for q, a in enumerate(args)]).double()
                        * dy.view(shape).double()).sum()) for sign in (1, -1)]
        slope, want = (s[0] - s[1]) / (2 * h), float((grads[i].double() * v.double()).sum())
        scale = float((grads[i].double() * v.double()).abs().sum())
        assert abs(slope - want) < 2e-3 * scale, (i, slope, want)


def test_another_stream_and_graph_replay():
    """A captured forward and backward whose offsets and rows change between replays, beside eager calls."""
    from mace_onegpu.group_norm import group_norm
    g = torch.Generator().manual_seed(3)
    x, w, b, dy = (t.cuda() for t in _inputs(3000, 64, torch.float32, torch.float32, 4))
    o = torch.tensor([0, 10, 2000, 2000, 2990], dtype=torch.int32).cuda()
    want = group_norm(x, 4, w, b, offsets=o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = group_norm(x, 4, w, b, offsets=o)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    xs, os_ = x.clone().requires_grad_(), o.clone()

    def step():
        y = group_norm(xs, 4, w, b, activation="silu", offsets=os_)
        return y.detach(), torch.autograd.grad(y, xs, dy)[0]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys, dxs = step()
    for cut in (2500, 7, 1200):
        with torch.no_grad():
            xs.copy_(torch.randn(3000, 64, generator=g))
        os_.copy_(torch.tensor([0, cut, cut, 2600, 3000], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        y, dx = step()
        assert torch.equal(ys, y) and torch.equal(dxs, dx)


def test_refusals():
    from mace_onegpu.group_norm import group_norm
    x, w = torch.randn(2, 6, 32).cuda(), torch.ones(32).cuda()
    o = torch.tensor([0, 12]).cuda()
    for error, call in [(TypeError, lambda: group_norm(x.cpu(), 4)),
                        (TypeError, lambda: group_norm(x.double(), 4)),
                        (ValueError, lambda: group_norm(x[0, 0], 4)),
                        (ValueError, lambda: group_norm(x, 5)),
                        (ValueError, lambda: group_norm(x, 0)),
                        (ValueError, lambda: group_norm(x, 4, w[:31])),
                        (TypeError, lambda: group_norm(x, 4, w.half())),
                        (TypeError, lambda: group_norm(x.half(), 4, w, w.half())),
                        (ValueError, lambda: group_norm(x, 4, activation="relu")),
                        (ValueError, lambda: group_norm(x, 4, offsets=o)),
                        (ValueError, lambda: group_norm(x[0], 4, offsets=o[:1])),
                        (TypeError, lambda: group_norm(x[0], 4, offsets=o.float())),
                        (TypeError, lambda: group_norm(x[0], 4, offsets=o.cpu())),
                        (ValueError, lambda: group_norm(torch.randn(1, 2, 4097).cuda(), 1))]:
        with pytest.raises(error):
            call()
    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(group_norm(xg, 4).square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        dx.sum().backward()
