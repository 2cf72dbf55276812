"""orthogonalize against the iteration in 64 bits on the same (rounded) inputs, and the Muon optimizer.

Tolerance, by matrix in the Frobenius norm.  An operand of a product is off by r = 2^-22 of itself (two float16 parts;
2^-11 for bfloat16's one part), every result of n products by 3 n u of the products' magnitudes, u = 2^-24.  A step
X' = a X + B X, B = b A + c A A, A = X X^T, then adds an error of at most

    noise = 2 r |B| |X|_F + |X| (r |B|_F + (|b| + 2 |c| |A|) dA + |c| n u ..) + 4 u |X'|_F,
    dA = 2 r |X| |X|_F + r |A|_F

(|.| spectral), sums' terms included below; and an error present before a step grows by at most max(a, max |p'|) over the
singular values, p(s) = a s + b s^3 + c s^5.  Rounding to the type adds half a unit in the last place of each entry."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
C = (3.4445, -4.7750, 2.0315)


def _matrices(E, m, n, dtype, seed, scale=0.01):
    g = torch.Generator().manual_seed(seed)
    r = max(1, min(m, n) // 8)
    strong = torch.bmm(torch.randn(E, m, r, generator=g) * torch.exp(torch.randn(E, 1, r, generator=g)),
                       torch.randn(E, r, n, generator=g)) / r ** 0.5
    return (scale * (strong + 0.3 * torch.randn(E, m, n, generator=g))).to(dtype)


def _reference(m, dtype, steps=5, coefficients=C, eps=1e-7):
    """One matrix in 64 bits: the result and the bound of its error."""
    x = m.double()
    tall = x.shape[0] > x.shape[1]
    x = x.T.contiguous() if tall else x
    x = x / (torch.linalg.matrix_norm(x) + eps)
    fro = lambda t: float(torch.linalg.matrix_norm(t))  # noqa: E731
    top = lambda t: float(torch.linalg.matrix_norm(t, 2))  # noqa: E731
    r = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22
    n = max(x.shape)
    err = 4 * U * fro(x)
    a, b, c = coefficients
    for _ in range(steps):
        A = x @ x.T
        B = b * A + c * A @ A
        s, f, sA = top(x), fro(x), top(A)
        dA = 2 * r * s * f + r * fro(A) + 3 * n * U * fro(x.abs() @ x.abs().T)
        dB = (r * fro(B) + (abs(b) + 2 * abs(c) * sA) * dA
              + abs(c) * (2 * r * sA * fro(A) + 3 * n * U * fro(A.abs() @ A.abs())))
        new = a * x + B @ x
        noise = 2 * r * top(B) * f + s * dB + 3 * n * U * fro(B.abs() @ x.abs()) + 4 * U * (a * f + fro(new))
        t = torch.linspace(0, s, 1000, dtype=torch.float64)
        gain = max(abs(a), float((a + 3 * b * t ** 2 + 5 * c * t ** 4).abs().max()))
        err = gain * err + noise
        x = new
    out = x.T if tall else x
    return out, err + HALF_ULP[dtype] * fro(out)


def _plain(m):
    x = m.float()
    tall = x.shape[0] > x.shape[1]
    x = x.T.contiguous() if tall else x
    x = x / (x.double().norm().float() + 1e-7)
    for _ in range(5):
        A = x @ x.T
        x = C[0] * x + (C[1] * A + C[2] * A @ A) @ x
    return x.T if tall else x


SIZES = [(1, 1, 1), (3, 1, 9), (2, 16, 16), (4, 30, 30), (2, 64, 64), (3, 65, 33), (8, 128, 128), (2, 201, 137),
         (2, 137, 201), (1, 300, 128), (1, 128, 1000), (1, 513, 260), (2, 7, 700)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,m,n", SIZES)
def test_against_64_bits(E, m, n, dtype):
    from mace_onegpu.muon import orthogonalize
    M = _matrices(E, m, n, dtype, E + m + n)
    got = orthogonalize(M.cuda())
    assert got.shape == M.shape and got.dtype == dtype and torch.equal(got, orthogonalize(M.cuda()))
    for e in range(E):
        want, bound = _reference(M[e], dtype)
        err = float(torch.linalg.matrix_norm(got[e].double().cpu() - want))
        assert err <= bound, (e, err, bound)
        if dtype == torch.float32:      # as near as float32 arithmetic comes
            plain = float(torch.linalg.matrix_norm(_plain(M[e]).double() - want))
            assert err <= 8 * plain + 2.0 ** -22 * float(torch.linalg.matrix_norm(want)), (e, err, plain)
        assert torch.equal(got[e], orthogonalize(M[e:e + 1].cuda())[0])     # whatever stands beside it


def test_singular_values_and_vectors():
    from mace_onegpu.muon import orthogonalize
    M = _matrices(1, 96, 160, torch.float32, 1)[0]
    u, s, v = torch.linalg.svd(M.double(), full_matrices=False)
    out = orthogonalize(M.cuda()).double().cpu()
    t = u.T @ out @ v.T
    d = torch.diagonal(t)
    assert float((t - torch.diag(d)).abs().max()) < 1e-4            # the singular vectors stay
    assert bool((d[s > 0.01 * s[0]] > 0.6).all()) and float(d.max()) < 1.3


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1.0, 1e18, 1e30])
def test_scale_of_the_matrix_does_not_matter(scale):
    from mace_onegpu.muon import orthogonalize
    M = _matrices(2, 40, 70, torch.float32, 2, scale=1.0)
    got = orthogonalize((M.double() * scale).float().cuda(), eps=0.0)
    want = orthogonalize(M.cuda(), eps=0.0)
    assert float((got - want).abs().max()) < 1e-4 * float(want.abs().max())


def test_steps_and_coefficients():
    from mace_onegpu.muon import orthogonalize
    M = _matrices(2, 50, 60, torch.float32, 3)
    none = orthogonalize(M.cuda(), steps=0)
    want = M.double() / (torch.linalg.matrix_norm(M.double())[:, None, None] + 1e-7)
    assert float((none.double().cpu() - want).abs().max()) <= 2 * U * float(want.abs().max())
    each = [(3.0, -4.0, 2.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375)]
    got = orthogonalize(M.cuda(), steps=3, coefficients=each)
    x = want
    for a, b, c in each:
        A = x @ x.mT.contiguous()
        x = a * x + (b * A + c * A @ A) @ x
    assert float((got.double().cpu() - x).abs().max()) < 1e-5 * float(x.abs().max())
    # more steps than one launch takes: the cubic iteration, whose errors only shrink (its slope stays below 1.5)
    for steps in (16, 17, 25):
        got = orthogonalize(M.cuda(), steps=steps, coefficients=(1.5, -0.5, 0.0))
        x = want
        for _ in range(steps):
            x = 1.5 * x - 0.5 * (x @ x.mT.contiguous()) @ x
        assert float((got.double().cpu() - x).abs().max()) < 2e-4 * float(x.abs().max())


def test_batches_strides_and_odd_matrices():
    from mace_onegpu.muon import orthogonalize
    M = _matrices(6, 24, 40, torch.float32, 4).cuda()
    want = orthogonalize(M)
    assert torch.equal(orthogonalize(M.view(2, 3, 24, 40)), want.view(2, 3, 24, 40))
    assert torch.equal(orthogonalize(M[0]), want[0])
    assert torch.equal(orthogonalize(M.mT.contiguous().mT), want)
    assert torch.equal(orthogonalize(M[::2]), want[::2])
    wide = torch.zeros(6, 24, 50, device="cuda")
    wide[:, :, 3:43] = M
    assert torch.equal(orthogonalize(wide[:, :, 3:43]), want)
    assert orthogonalize(M[:0]).shape == (0, 24, 40)
    bad = M.clone()
    bad[1], bad[3, 2, 5], bad[4, 0, 0] = 0.0, float("nan"), float("inf")
    got = orthogonalize(bad)
    assert not got[1].any() and got[3].isnan().all() and got[4].isnan().all()
    for e in (0, 2, 5):
        assert torch.equal(got[e], want[e])
    assert torch.equal(orthogonalize(torch._neg_view(-M)), want)


def test_another_stream_and_graph_replay():
    from mace_onegpu.muon import orthogonalize
    M = _matrices(3, 100, 72, torch.bfloat16, 5).cuda()
    want = orthogonalize(M)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = orthogonalize(M)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    s = M.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = orthogonalize(s)
    for seed in (6, 7, 8):
        s.copy_(_matrices(3, 100, 72, torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, orthogonalize(s))


def test_refusals():
    from mace_onegpu.muon import Muon, orthogonalize
    M = torch.randn(2, 8, 8, device="cuda")
    for error, call in [(TypeError, lambda: orthogonalize(M.cpu())), (TypeError, lambda: orthogonalize(M.double())),
                        (ValueError, lambda: orthogonalize(M[0, 0])), (ValueError, lambda: orthogonalize(M[:, :0])),
                        (ValueError, lambda: orthogonalize(M, steps=-1)),
                        (ValueError, lambda: orthogonalize(M, eps=-1.0)),
                        (ValueError, lambda: orthogonalize(M, eps=float("nan"))),
                        (ValueError, lambda: orthogonalize(M, steps=2, coefficients=[C])),
                        (ValueError, lambda: orthogonalize(M, coefficients=(1.0, 2.0))),
                        (ValueError, lambda: orthogonalize(torch.zeros(1, 65537, device="cuda"))),
                        (RuntimeError, lambda: orthogonalize(M.clone().requires_grad_())),
                        (ValueError, lambda: Muon([torch.nn.Parameter(M[0, 0].clone())])),
                        (ValueError, lambda: Muon([torch.nn.Parameter(M.clone())], momentum=1.0))]:
        with pytest.raises(error):
            call()
    with torch.no_grad():
        assert orthogonalize(M.clone().requires_grad_()).shape == M.shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_steps(nesterov, dtype):
    """Three steps against the rule written out; parameters without a gradient stay; the state is saved and loaded."""
    from mace_onegpu.muon import Muon, orthogonalize
    p = [torch.nn.Parameter(_matrices(4, 24, 40, dtype, 10).cuda()),
         torch.nn.Parameter(_matrices(1, 30, 10, dtype, 11)[0].cuda()),
         torch.nn.Parameter(torch.ones(3, 3, dtype=dtype, device="cuda"))]
    opt = Muon(p, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    want = [q.detach().clone() for q in p]
    buf = [torch.zeros_like(q, dtype=torch.float32) for q in want]
    for step in range(3):
        for i in range(2):
            g = _matrices(*((4, 24, 40) if i == 0 else (1, 30, 10)), dtype, 20 + 2 * step + i).cuda().view(p[i].shape)
            p[i].grad = g
            buf[i] = buf[i] * 0.9 + g.float()
            u = g.float() + 0.9 * buf[i] if nesterov else buf[i]
            want[i] = (want[i] * (1 - 0.02 * 0.1)
                       - (0.02 * 0.2 * max(want[i].shape[-2:]) ** 0.5) * orthogonalize(u.to(dtype)))
        opt.step()
        if step == 0:
            saved = opt.state_dict()
            opt = Muon(p, lr=0.5)
            opt.load_state_dict(saved)
    for i in range(2):
        # a few roundings of the type a step; u of bfloat16 may round to its other neighbour after another order of sums
        assert float((p[i].detach().float() - want[i].float()).abs().max()) < (1e-5 if dtype == torch.float32 else 2e-2)
        assert opt.state[p[i]]["momentum_buffer"].dtype == torch.float32
    assert torch.equal(p[2].detach(), torch.ones_like(p[2]))
