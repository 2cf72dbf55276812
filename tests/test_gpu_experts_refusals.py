"""Arguments that layer_norm, route, plan_experts and expert_linear refuse, each before a launch."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def test_layer_norm():
    from mace_onegpu.layer_norm import layer_norm
    x = _z(3, 8)
    for args, err, match in [((x.double(),), TypeError, "float32, bfloat16 or float16"),
                             ((x.long(),), TypeError, "float32, bfloat16 or float16"),
                             ((x, _z(7)), ValueError, r"weight must be \[8\]"),
                             ((x, _z(8), _z(1, 8)), ValueError, r"bias must be \[8\]"),
                             ((x, _z(8, dtype=torch.float16)), TypeError, "weight must be"),
                             ((x.bfloat16(), _z(8), _z(8, dtype=torch.bfloat16)), TypeError, "one type"),
                             ((x, torch.zeros(8)), TypeError, "weight must be a GPU tensor"),
                             ((_z(3, 0),), ValueError, "D > 0"), ((_z(2, 16385),), ValueError, "16384")]:
        with pytest.raises(err, match=match):
            layer_norm(*args)


def test_route():
    from mace_onegpu.experts import route
    x = _z(3, 8)
    for args, kw, err, match in [((x[0], 2), {}, ValueError, r"\[rows, experts\]"),
                                 ((x, 0), {}, ValueError, "k must be"),
                                 ((x, 9), {}, ValueError, "k must be"), ((_z(3, 64), 33), {}, ValueError, "k must be"),
                                 ((_z(3, 1025), 2), {}, ValueError, "1024 experts"),
                                 ((x, 2), dict(scoring="relu"), ValueError, "scoring"),
                                 ((x, 2), dict(groups=3), ValueError, "groups must divide"),
                                 ((_z(3, 130), 2), dict(groups=65), ValueError, "at most 64"),
                                 ((x, 2), dict(groups=4, top_groups=5), ValueError, "top_groups"),
                                 ((x, 2), dict(scale=0), ValueError, "scale"),
                                 ((x, 2), dict(scale=float("inf")), ValueError, "scale"),
                                 ((x, 2), dict(bias=_z(7)), ValueError, r"bias must be \[8\]"),
                                 ((x, 2), dict(bias=_z(8, dtype=torch.float16)), TypeError, "bias must be float32"),
                                 ((x.double(), 2), {}, TypeError, "logits must be float32")]:
        with pytest.raises(err, match=match):
            route(*args, **kw)


def test_plan_and_products():
    from mace_onegpu.experts import expert_linear, plan_experts
    e = _z(4, 2, dtype=torch.int32)
    for args, err, match in [((e.float(), 3), TypeError, "int32 or int64"), ((e[0], 3), ValueError, r"\[rows, k\]"),
                             ((e, 0), ValueError, "n_experts"), ((e, 1025), ValueError, "n_experts")]:
        with pytest.raises(err, match=match):
            plan_experts(*args)
    plan, x, w, g = plan_experts(e, 3), _z(4, 8), _z(3, 8, 5), _z(4, 2)
    for args, err, match in [((x, w.half(), plan, g), TypeError, "weight must be"),
                             ((x, w, e, g), TypeError, "ExpertPlan"),
                             ((x[0], w, plan, g), ValueError, "x must be"), ((x[:3], w, plan, g), ValueError, "3 rows"),
                             ((x, w[:2], plan, g), ValueError, "weight must be"), ((x[:, :7], w, plan, g), ValueError,
                                                                                    "weight must be"),
                             ((x, w[:, :, :0], plan, g), ValueError, "weight must be"),
                             ((x[:, None][:, :0], w, plan, g), ValueError, "no components"),
                             ((x, w, plan, g.half()), TypeError, "gates must be float32"),
                             ((x, w, plan, g[:, :1]), ValueError, "gates must be")]:
        with pytest.raises(err, match=match):
            expert_linear(*args)


def test_second_derivatives_are_refused():
    """Gradients are taken once: differentiating them again raises, it does not pass them off as constants."""
    from mace_onegpu.experts import expert_linear, plan_experts, route
    from mace_onegpu.layer_norm import layer_norm
    x = torch.randn(5, 8, generator=torch.Generator().manual_seed(0)).cuda().requires_grad_()
    w = torch.randn(4, 8, 8, generator=torch.Generator().manual_seed(1)).cuda()
    plan = plan_experts(torch.randint(0, 4, (5, 2)).cuda(), 4)
    for f in (lambda: layer_norm(x), lambda: route(x, 2)[0], lambda: expert_linear(x, w, plan)):
        (dx,) = torch.autograd.grad(f().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once only"):
            dx.square().sum().backward()


def test_each_gradient_alone():
    """Only some inputs ask for a gradient: it is the same one as when all do."""
    from mace_onegpu.experts import expert_linear, plan_experts
    from mace_onegpu.layer_norm import layer_norm
    g = torch.Generator().manual_seed(2)
    x, w, b = (torch.randn(*s, generator=g).cuda() for s in ((30, 24), (24,), (24,)))
    blocks, gates = torch.randn(4, 24, 16, generator=g).cuda(), torch.rand(30, 2, generator=g).cuda()
    plan = plan_experts(torch.randint(0, 4, (30, 2), generator=g).cuda(), 4)
    for f, args in ((layer_norm, (x, w, b)), (lambda a, c, d: expert_linear(a, c, plan, d), (x, blocks, gates))):
        every = [t.clone().requires_grad_() for t in args]
        want = torch.autograd.grad(f(*every).square().sum(), every)
        for i in range(3):
            one = [t.clone().requires_grad_(q == i) for q, t in enumerate(args)]
            (got,) = torch.autograd.grad(f(*one).square().sum(), one[i])
            assert torch.equal(got, want[i])
    bias = b.clone().requires_grad_()
    (got,) = torch.autograd.grad(layer_norm(x, None, bias).sum(), bias)       # a bias without a weight
    assert torch.equal(got, torch.full_like(b, 30.0))
