"""Gradients under saved-tensor hooks that give back other strides: the same bits as without hooks.  Another size or type
is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _transposed(t):
    """the same values with the axes laid out in the opposite order"""
    n = t.dim()
    back = tuple(range(n))[::-1]
    return t.permute(back).contiguous().permute(back)


def _spread(t):
    """the same values as every second one of a larger array (a row distance that was not saved)"""
    wide = torch.zeros(*t.shape[:-1], 2 * t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


def _hooks(which):
    if which == "cpu":
        return torch.autograd.graph.save_on_cpu()
    return torch.autograd.graph.saved_tensors_hooks(which, lambda t: t)


def _norm_calls(dtype):
    from mace_onegpu.layer_norm import layer_norm
    g = torch.Generator().manual_seed(1)
    for rows, D in ((1, 8), (77, 24), (500, 128), (33, 1031), (9, 5000)):
        h = torch.randn(rows, 4, D, generator=g).to(dtype).cuda()
        w, b = torch.randn(D, generator=g).to(dtype).cuda(), torch.randn(D, generator=g).to(dtype).cuda()
        yield (lambda x, w, b: layer_norm(x[:, 0], w, b)), (h, w, b)             # a strided slice: read in place
        yield (lambda x, w, b: layer_norm(x, w, b)), (h, w, b)
        yield (lambda x: layer_norm(x[:, 2])), (h,)


def _route_calls(dtype):
    from mace_onegpu.experts import route
    g = torch.Generator().manual_seed(2)
    for T, E, k in ((1, 4, 2), (300, 16, 2), (64, 89, 3)):
        x = torch.randn(T, E + 5, generator=g).to(dtype).cuda()
        for kw in (dict(), dict(scoring="sigmoid"), dict(renormalize=False)):
            yield (lambda x, E=E, k=k, kw=kw: route(x[:, :E], k, **kw)[0]), (x,)


def _linear_calls(dtype):
    from mace_onegpu.experts import expert_linear, plan_experts
    g = torch.Generator().manual_seed(3)
    for T, M, D, F, E, k in ((3, 1, 32, 24, 4, 2), (400, 3, 64, 72, 5, 3), (500, 1, 128, 64, 3, 1),
                             (9000, 1, 128, 128, 2, 2)):
        x, w = torch.randn(T, M + 1, D, generator=g).to(dtype).cuda(), torch.randn(E, D, F, generator=g).to(dtype).cuda()
        e = torch.randint(-1, E, (T, k), generator=g, dtype=torch.int32).cuda()
        gates = torch.rand(T, k, generator=g).cuda()
        plan = plan_experts(e, E)
        yield (lambda x, w, q, plan=plan: expert_linear(x[:, 1:], w, plan, q)), (x, w, gates)
        yield (lambda x, w, plan=plan: expert_linear(x[:, 0], w, plan)), (x, w)


@pytest.mark.parametrize("hook", ["cpu", _transposed, _spread])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("calls", [_norm_calls, _route_calls, _linear_calls])
def test_same_gradients(calls, dtype, hook):
    for f, args in calls(dtype):
        args = [t.requires_grad_() for t in args]
        y = f(*args)
        dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(4)).to(y.dtype).cuda()
        want = torch.autograd.grad(y, args, dy)
        with _hooks(hook):
            z = f(*args)
        got = torch.autograd.grad(z, args, dy)
        assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("calls", [_norm_calls, _route_calls, _linear_calls])
def test_other_sizes_and_types_are_refused(calls):
    f, args = next(iter(calls(torch.float32)))
    args = [t.requires_grad_() for t in args]
    for hook in (lambda t: t.double(), lambda t: t[..., :0], lambda t: t.reshape(-1, 1), lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(hook, lambda t: t):
            y = f(*args)
        with pytest.raises(RuntimeError, match="was saved for the backward as"):
            torch.autograd.grad(y, args, torch.ones_like(y))
