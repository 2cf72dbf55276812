"""layer_norm and its gradients against the formula in 64 bits on the same (rounded) inputs.

Tolerances, element by element, u = 2^-24: a sum of n values in lanes and trees has at most C = 32 + 10 roundings on any
path (32 values a lane, 1024 lanes), so the mean is off by at most C u max|x| and, scaled by rstd and w, so is y; the
other operations add less than 16 u of their terms.  Rounding to the output's type adds half a unit in its last place. 
dw and db: the same with sums over rows (a lane's rows, then up to 1024 partial sums in trees and 16 in a row)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
CHAIN = 64


def _inputs(rows, D, dtype, p_dtype, seed, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, D, generator=g) * torch.exp(0.5 * torch.randn(rows, 1, generator=g)) + offset).to(dtype)
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(p_dtype)
    b = (0.2 * torch.randn(D, generator=g)).to(p_dtype)
    dy = torch.randn(rows, D, generator=g).to(dtype)
    return x, w, b, dy


def _reference(x, w, b, dy, eps):
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    mu = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + eps)
    h = (x - mu) * r
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return dict(y=h * w + b, dx=dx, dw=(dy * h).sum(0), db=dy.sum(0), h=h, r=r, g=g)


def _bounds(x, w, b, dy, ref, dtype, p_dtype, rows):
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    h, r, g = ref["h"], ref["r"], ref["g"]
    dh = U * (CHAIN * x.abs().amax(1, keepdim=True) * r + CHAIN * h.abs())       # error of the normalised x
    ag, agh = g.abs().mean(1, keepdim=True), (g * h).abs().mean(1, keepdim=True)
    gdh = (g.abs() * dh).mean(1, keepdim=True)
    dx = r * (CHAIN * U * (g.abs() + ag + h.abs() * agh) + dh * agh + h.abs() * gdh)
    chain = rows / 1024 + 96 + 32
    return dict(y=dh * w.abs() + 16 * U * ((h * w).abs() + b.abs()) + HALF_ULP[dtype] * ref["y"].abs(),
                dx=dx + HALF_ULP[dtype] * ref["dx"].abs(),
                dw=chain * U * (dy * h).abs().sum(0) + (dy.abs() * dh).sum(0) + HALF_ULP[p_dtype] * ref["dw"].abs(),
                db=chain * U * dy.abs().sum(0) + HALF_ULP[p_dtype] * ref["db"].abs())


def _tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 1e-37     # half the least subnormal


def _check(got, ref, bound, tiny):
    for name, t in got.items():
        err = (t.detach().double().cpu() - ref[name]).abs()
        assert bool((err <= bound[name] + tiny).all()), (name, float((err - bound[name]).max()))


@pytest.mark.parametrize("dtype,p_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                           (torch.float16, torch.float16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 2), (5, 17), (257, 64), (1000, 96), (37, 128), (19, 257), (33, 1000),
                                    (9, 1031), (130, 2048), (7, 4095), (5, 5000), (3, 8192), (2, 16383), (3001, 8)])
def test_forward_and_gradients(rows, D, dtype, p_dtype):
    from mace_onegpu.layer_norm import layer_norm
    x, w, b, dy = _inputs(rows, D, dtype, p_dtype, rows + D)
    eps = 1e-5
    ref = _reference(x, w, b, dy, eps)
    bound = _bounds(x, w, b, dy, ref, dtype, p_dtype, rows)
    xg, wg, bg = (t.cuda().requires_grad_() for t in (x, w, b))
    y = layer_norm(xg, wg, bg, eps)
    assert y.dtype == dtype and y.shape == x.shape
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), dy.cuda())
    assert (dx.dtype, dw.dtype, db.dtype) == (dtype, p_dtype, p_dtype)
    _check(dict(y=y, dx=dx, dw=dw, db=db), ref, bound, _tiny(dtype))
    with torch.no_grad():
        assert torch.equal(layer_norm(xg, wg, bg, eps), y)


def test_many_rows_of_a_radial_layer():
    from mace_onegpu.layer_norm import layer_norm
    rows, D = 100003, 64
    x, w, b, dy = _inputs(rows, D, torch.float32, torch.float32, 5)
    ref = _reference(x, w, b, dy, 1e-5)
    bound = _bounds(x, w, b, dy, ref, torch.float32, torch.float32, rows)
    xg, wg, bg = (t.cuda().requires_grad_() for t in (x, w, b))
    grads = [torch.autograd.grad(layer_norm(xg, wg, bg), (xg, wg, bg), dy.cuda()) for _ in range(2)]
    for a, c in zip(*grads):
        assert torch.equal(a, c)           # no order of sums changes from run to run
    _check(dict(zip(("dx", "dw", "db"), grads[0])), ref, bound, 1e-37)


def test_strided_rows_and_leading_axes():
    from mace_onegpu.layer_norm import layer_norm
    g = torch.Generator().manual_seed(1)
    feats = torch.randn(33, 4, 128, generator=g).cuda()
    w, b = torch.randn(128, generator=g).cuda(), torch.randn(128, generator=g).cuda()
    whole = layer_norm(feats, w, b)
    assert torch.equal(layer_norm(feats[:, 0], w, b), whole[:, 0])
    assert torch.equal(layer_norm(feats[::2, 1:3], w, b), whole[::2, 1:3])
    assert torch.equal(layer_norm(feats.reshape(-1, 128).t().contiguous().t(), w, b), whole.view(-1, 128))
    cut = feats.view(33, 512)[:, 1:100]                       # rows that start off any 16-byte boundary
    assert torch.equal(layer_norm(cut, w[:99], b[:99]), layer_norm(cut.contiguous(), w[:99], b[:99]))
    x = feats[:, 0].detach().requires_grad_()
    (dx,) = torch.autograd.grad(layer_norm(x, w, b).sum(), x)          # an expanded cotangent
    (dx1,) = torch.autograd.grad(layer_norm(x, w, b), x, torch.ones(33, 128, device="cuda"))
    assert torch.equal(dx, dx1)
    one = layer_norm(feats[:1, 0].expand(5, 128), w, b)
    assert torch.equal(one, whole[:1, 0].expand(5, 128))


def test_without_weight_or_bias_and_module():
    from mace_onegpu.layer_norm import LayerNorm, layer_norm
    g = torch.Generator().manual_seed(2)
    x = torch.randn(50, 96, generator=g).cuda()
    w = torch.randn(96, generator=g).cuda()
    one, zero = torch.ones(96, device="cuda"), torch.zeros(96, device="cuda")
    assert torch.equal(layer_norm(x), layer_norm(x, one, zero))
    assert torch.equal(layer_norm(x, w), layer_norm(x, w, zero))
    m = LayerNorm(96, device="cuda")
    assert torch.equal(m(x), layer_norm(x))
    m(x).square().sum().backward()
    assert m.weight.grad.shape == (96,) and m.bias.grad.shape == (96,)
    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(layer_norm(xg).square().sum(), xg)
    assert float(dx.abs().max()) < 1e-3          # sum of squares of a norm is constant up to eps


def test_no_rows_and_constant_and_non_finite_rows():
    from mace_onegpu.layer_norm import layer_norm
    w = torch.ones(40, device="cuda", requires_grad=True)
    b = torch.ones(40, device="cuda", requires_grad=True)
    x = torch.empty(0, 40, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    assert y.shape == (0, 40)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 40, device="cuda"))
    assert dx.shape == (0, 40) and not dw.any() and not db.any()
    x = torch.full((3, 40), 7.0, device="cuda")
    x[1, 5], x[2, 39] = float("nan"), float("inf")
    with torch.no_grad():
        y = layer_norm(x, w, b)
    assert torch.equal(y[0], b) and y[1:].isnan().all()


@pytest.mark.parametrize("D", [64, 1000])
def test_gradient_against_differences(D):
    """<grad, v> against (f(x + h v) - f(x - h v)) / 2 h, f summed in 64 bits: off by O(h^2) and roundings of f over
    h."""
    from mace_onegpu.layer_norm import layer_norm
    x, w, b, dy = (t.cuda() for t in _inputs(11, D, torch.float32, torch.float32, D))
    g = torch.Generator().manual_seed(9)
    args = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*args), args, dy)
    h = 1e-2
    for i in range(3):
        v = torch.randn(args[i].shape, generator=g).cuda()
        with torch.no_grad():
            f = [float((layer_norm(*[a + s * h * v if q == i else a for q, a in enumerate(args)]).double()
                        * dy.double()).sum()) for s in (1, -1)]
        slope, want = (f[0] - f[1]) / (2 * h), float((grads[i].double() * v.double()).sum())
        scale = float((grads[i].double() * v.double()).abs().sum())
        assert abs(slope - want) < 2e-3 * scale, (i, slope, want)


def test_another_stream_and_graph_replay():
    from mace_onegpu.layer_norm import layer_norm
    g = torch.Generator().manual_seed(3)
    x, w, b, dy = (t.cuda() for t in _inputs(300, 128, torch.float32, torch.float32, 4))
    want = layer_norm(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer_norm(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    xs = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        with torch.cuda.graph(graph):
            ys = layer_norm(xs, w, b)
    for _ in range(3):
        xs.copy_(torch.randn(300, 128, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ys, layer_norm(xs, w, b))
