"""Tensors whose memory does not hold their values: lazily negated views give the results of the values, also as a
cotangent; fake, wrapped and zero tensors have no memory and are refused before a launch."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls():
    from mace_onegpu.experts import expert_linear, plan_experts, route
    from mace_onegpu.layer_norm import layer_norm
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    plan = plan_experts(torch.randint(0, 4, (30, 2), generator=g).cuda(), 4)
    yield layer_norm, [r(30, 24), r(24), r(24)]
    yield (lambda x, b: route(x, 2, bias=b)[0]), [r(30, 8), r(8)]
    yield (lambda x, w, q: expert_linear(x, w, plan, q)), [r(30, 24), r(4, 24, 16), r(30, 2)]


def _negated(t):
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


def test_negated_views():
    for f, args in _calls():
        want = f(*args)
        for i in range(len(args)):
            assert torch.equal(f(*[_negated(t) if q == i else t for q, t in enumerate(args)]), want)
    from mace_onegpu.experts import plan_experts
    e = torch.randint(0, 4, (30, 2), generator=torch.Generator().manual_seed(1)).cuda()
    for experts in (e, e.int()):
        assert torch.equal(plan_experts(_negated(experts), 4).counts, plan_experts(experts, 4).counts)


def test_negated_cotangents():
    for f, args in _calls():
        args = [t.requires_grad_() for t in (args[:1] if len(args) == 2 else args)] + args[1:2] * (len(args) == 2)
        leaves = [t for t in args if t.requires_grad]
        y = f(*args)
        dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).cuda()
        want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        got = torch.autograd.grad(y, leaves, _negated(dy))
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_imaginary_part_of_a_conjugate():
    from mace_onegpu.layer_norm import layer_norm
    z = torch.randn(9, 16, dtype=torch.complex64, generator=torch.Generator().manual_seed(3)).cuda()
    x = z.conj().imag
    assert x.is_neg() and torch.equal(layer_norm(x), layer_norm(x.resolve_neg()))


class _Wrapped(torch.Tensor):
    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise RuntimeError("not to be reached by the kernels")


def test_tensors_without_memory_are_refused():
    zero = lambda t: torch._efficientzerotensor(t.shape, device="cuda", dtype=t.dtype)  # noqa: E731
    for f, args in _calls():
        for i in range(len(args)):
            for fake in (zero, _Wrapped):
                with pytest.raises((TypeError, RuntimeError)):
                    f(*[fake(t) if q == i else t for q, t in enumerate(args)])
    torch.cuda.synchronize()


def test_fake_tensors_are_refused():
    from mace_onegpu.layer_norm import layer_norm
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(4, 8, device="cuda")
        with pytest.raises((TypeError, RuntimeError)):
            layer_norm(x)
