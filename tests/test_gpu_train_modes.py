"""Group norm, linear cross entropy and orthogonalisation on tensors that are not plain: dual tensors, traces, negated
views, tensors without memory, saved-tensor hooks, inference mode, and rows whose offsets pass 2^31 or 2^32 elements."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def _calls(dtype=torch.float32):
    from mace_onegpu.cross_entropy import linear_cross_entropy
    from mace_onegpu.group_norm import group_norm
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    y = torch.randint(0, 40, (30,), generator=g).cuda()
    o = torch.tensor([0, 7, 7, 28]).cuda()
    yield "group_norm", lambda x, w, b: group_norm(x, 4, w, b, activation="silu"), [r(3, 10, 24), r(24), r(24)]
    yield "group_norm", lambda x, w, b: group_norm(x, 4, w, b, activation="gelu", offsets=o), [r(30, 24), r(24), r(24)]
    yield "linear_cross_entropy", lambda x, w: linear_cross_entropy(x, w, y, reduction="none"), [r(30, 24), r(40, 24)]
    yield "linear_cross_entropy", lambda x, w: linear_cross_entropy(x, w, y[:5]), [r(5, 24), r(40, 24)]


def _ortho(x):
    from mace_onegpu.muon import orthogonalize
    return orthogonalize(x)


def test_dual_tensors_and_traces():
    for name, f, args in [*_calls(), ("orthogonalize", _ortho, [torch.randn(2, 6, 9).cuda()])]:
        for i in range(len(args)):
            with fwAD.dual_level():
                mixed = [fwAD.make_dual(t, torch.ones_like(t)) if q == i else t for q, t in enumerate(args)]
                with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
                    f(*mixed)
        with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
            torch.jit.trace(f, tuple(args))


def _negated(t):
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


def test_negated_views_and_cotangents():
    for _, f, args in _calls():
        want = f(*args)
        for i in range(len(args)):
            assert torch.equal(f(*[_negated(t) if q == i else t for q, t in enumerate(args)]), want)
        leaves = [t.clone().requires_grad_() for t in args]
        y = f(*leaves)
        dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).cuda()
        one = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        two = torch.autograd.grad(y, leaves, _negated(dy))
        assert all(torch.equal(a, b) for a, b in zip(one, two))


class _Wrapped(torch.Tensor):
    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise RuntimeError("not to be reached by the kernels")


def test_tensors_without_memory_are_refused():
    zero = lambda t: torch._efficientzerotensor(t.shape, device="cuda", dtype=t.dtype)  # noqa: E731
    for _, f, args in [*_calls(), ("orthogonalize", _ortho, [torch.randn(2, 6, 9).cuda()])]:
        for i in range(len(args)):
            for fake in (zero, _Wrapped):
                with pytest.raises((TypeError, RuntimeError)):
                    f(*[fake(t) if q == i else t for q, t in enumerate(args)])
    torch.cuda.synchronize()


def _transposed(t):
    back = tuple(range(t.dim()))[::-1]
    return t.permute(back).contiguous().permute(back)


def _spread(t):
    if t.dim() == 0:
        return t
    wide = torch.zeros(*t.shape[:-1], 2 * t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_saved_tensor_hooks(dtype):
    for _, f, args in _calls(dtype):
        def grads(which):
            leaves = [t.clone().requires_grad_() for t in args]
            hooks = (torch.autograd.graph.save_on_cpu() if which == "cpu"
                     else torch.autograd.graph.saved_tensors_hooks(which, lambda t: t))
            with hooks:
                y = f(*leaves)
            return torch.autograd.grad(y, leaves, torch.ones_like(y))
        want = grads(lambda t: t)
        for which in (_transposed, _spread, "cpu"):
            assert all(torch.equal(a, b) for a, b in zip(want, grads(which))), which
        with pytest.raises(RuntimeError, match="was saved for the backward as"):
            grads(lambda t: t.double() if t.is_floating_point() else t)


def test_inference_mode():
    for _, f, args in [*_calls(), ("orthogonalize", _ortho, [torch.randn(2, 6, 9).cuda()])]:
        want = f(*args)
        with torch.inference_mode():
            assert torch.equal(f(*[t.clone() for t in args]), want)


def test_two_graphs_of_one_stream():
    """Their workspaces are their own: replayed in turn, with eager calls between."""
    graphs = []
    for _, f, args in [*_calls(), ("orthogonalize", _ortho, [torch.randn(2, 200, 300).cuda()])]:
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph):
            out = f(*args)
        graphs.append((graph, out, f, args))
    for _ in range(3):
        for graph, out, f, args in graphs:
            args[0].copy_(torch.randn_like(args[0]))
            graph.replay()
        for graph, out, f, args in graphs:
            with torch.no_grad():
                want = f(*args)
            torch.cuda.synchronize()
            assert torch.equal(out, want)


TAIL = 300


@pytest.mark.parametrize("ragged", [False, True])
def test_group_norm_far_rows(ragged):
    from mace_onegpu.group_norm import group_norm
    x = torch.zeros(140000, 4, 8192, dtype=torch.float16, device="cuda")
    assert x.numel() > 2 ** 32
    x[-TAIL:] = torch.randn(TAIL, 4, 8192, generator=torch.Generator().manual_seed(1)).half().cuda()
    o = torch.tensor([0, 140000 - TAIL, 140000 - TAIL + 13, 140000]).cuda() if ragged else None
    x = x[:, 3] if ragged else x[:, 3].view(1400, 100, 8192)
    x.requires_grad_()
    y = group_norm(x, 8, offsets=o)
    dy = torch.zeros(140000, 8192, dtype=torch.float16, device="cuda")
    dy[-TAIL:] = 0.5
    dy[-1] = 1.0
    (dx,) = torch.autograd.grad(y, x, dy.view(x.shape))
    small = x.detach().view(140000, 8192)[-TAIL:].clone()
    small = (small if ragged else small.view(3, 100, 8192)).requires_grad_()
    z = group_norm(small, 8, offsets=torch.tensor([0, 13, 300]).cuda() if ragged else None)
    (dz,) = torch.autograd.grad(z, small, dy[-TAIL:].view(small.shape).clone())
    # other blocks of rows and channels: sums in another order, two results on both sides of a rounding (2^-10), and of
    # dx, whose terms of up to 1 cancel, 64 roundings of float32
    for a, b in ((y, z), (dx, dz)):
        assert torch.allclose(a.detach().view(-1, 8192)[-TAIL:].float(), b.detach().view(-1, 8192).float(),
                              rtol=2.0 ** -10, atol=2e-5)


def test_cross_entropy_far_classes():
    """Weights of more than 2^31 elements: rows of the last classes, against float32 products of them."""
    from mace_onegpu.cross_entropy import linear_cross_entropy
    V, D = 530000, 4096
    w = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    assert w.numel() > 2 ** 31
    g = torch.Generator().manual_seed(2)
    w[-TAIL:] = (torch.randn(TAIL, D, generator=g) / 64).bfloat16().cuda()
    w.requires_grad_()
    for T in (1, 40):
        x = torch.randn(T, D, generator=g).bfloat16().cuda()
        y = (V - 1 - torch.randint(0, TAIL, (T,), generator=g)).cuda()
        loss = linear_cross_entropy(x, w, y, reduction="none")
        logits = x.double() @ w.detach()[-TAIL:].double().T.contiguous()
        # the other classes have logits of 0
        lse = torch.log(torch.exp(logits).sum(1) + (V - TAIL))
        want = lse - logits.gather(1, (y - (V - TAIL))[:, None]).squeeze(1)
        assert float((loss.detach().double() - want).abs().max()) < 1e-4
        (dw,) = torch.autograd.grad(loss.sum(), w)
        p = torch.exp(logits - lse[:, None])
        p[torch.arange(T), y - (V - TAIL)] -= 1
        ref = p.T.contiguous() @ x.double()
        # d rounded to bfloat16 (2^-8 of every term), and the result
        bound = 2.0 ** -8 * (p.abs().T.contiguous() @ x.double().abs() + ref.abs()) + 1e-5
        assert bool(((dw[-TAIL:].double() - ref).abs() <= bound).all())
        far = torch.exp(-lse)[:, None].T @ x.double()
        assert float((dw[12345].double() - far[0]).abs().max()) < 1e-6
        del dw


def test_orthogonalize_far_matrices():
    """A batch whose last matrix lies past 2^32 elements, in parts; no steps: the norms and the copies alone."""
    from mace_onegpu.muon import orthogonalize
    m = torch.zeros(3, 38000, 38000, dtype=torch.bfloat16, device="cuda")
    assert m.numel() > 2 ** 32
    m[2, -50:, -70:] = torch.randn(50, 70, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    out = orthogonalize(m, steps=0)
    want = m[2, -50:, -70:].double()
    want = want / (want.norm() + 1e-7)
    err = (out[2, -50:, -70:].double() - want).abs()
    assert bool((err <= 2.0 ** -8 * want.abs() + 1e-9).all()) and not out[:2].any() and not out[2, :-50].any()
