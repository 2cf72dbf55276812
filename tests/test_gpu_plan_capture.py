"""A plan made under graph capture, used outside its graph: every product after a replay follows the replay's experts, in
eager calls and in other graphs; before the first replay its lists are never taken from memory that holds nothing."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# pairs held, pairs in tiles of 16 bits, one choice, slots, few rows
CASES = [(40000, 2, 3, torch.float32), (280000, 2, 2, torch.bfloat16), (9000, 1, 6, torch.float32),
         (5000, 3, 8, torch.float16), (40, 2, 8, torch.float32)]


def _case(T, k, E, dtype):
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, 64, generator=g).to(dtype).cuda()
    w = torch.randn(E, 64, 64, generator=g).to(dtype).cuda()
    return g, x, w, torch.randn(T, E, generator=g).cuda()


def _captured(logits, k, E):
    from mace_onegpu.experts import plan_experts, route
    route(logits, k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gates, experts = route(logits, k)
        plan = plan_experts(experts, E)
    return graph, gates, plan


@pytest.mark.parametrize("T,k,E,dtype", CASES)
def test_eager_products_follow_the_replays(T, k, E, dtype):
    from mace_onegpu.experts import expert_linear, plan_experts, route
    g, x, w, logits = _case(T, k, E, dtype)
    graph, gates, plan = _captured(logits, k, E)
    for _ in range(3):
        logits.copy_(torch.randn(T, E, generator=g))
        graph.replay()
        want_gates, experts = route(logits, k)
        fresh = plan_experts(experts, E)
        assert torch.equal(plan.experts, experts) and torch.equal(gates, want_gates)
        for _ in range(2):
            a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
            y, z = expert_linear(a, b, plan, gates), expert_linear(a, b, fresh, want_gates)
            assert torch.equal(y, z)
            for p, q in zip(torch.autograd.grad(y.float().sum(), (a, b)), torch.autograd.grad(z.float().sum(), (a, b))):
                assert torch.equal(p, q)
        for name in ("offsets", "order", "counts"):
            assert torch.equal(getattr(plan, name), getattr(fresh, name))


@pytest.mark.parametrize("T,k,E,dtype", CASES)
def test_another_graph_follows_the_replays(T, k, E, dtype):
    from mace_onegpu.experts import expert_linear, plan_experts, route
    g, x, w, logits = _case(T, k, E, dtype)
    graph, gates, plan = _captured(logits, k, E)
    graph.replay()
    torch.cuda.synchronize()
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        y = expert_linear(x, w, plan, gates)
    for _ in range(3):
        logits.copy_(torch.randn(T, E, generator=g))
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        want_gates, experts = route(logits, k)
        assert torch.equal(y, expert_linear(x, w, plan_experts(experts, E), want_gates))


def test_before_the_first_replay():
    """The experts hold whatever their memory held, which the kernels check against the number of experts; the lists are
    sorted from them and never read from the graph's memory."""
    from mace_onegpu.experts import expert_linear
    for T, k, E, dtype in CASES:
        _, x, w, logits = _case(T, k, E, dtype)
        graph, gates, plan = _captured(logits, k, E)
        assert expert_linear(x, w, plan, gates).shape == (T, 64)
        n = int(plan.offsets[-1])
        assert 0 <= n <= T * k and int(plan.counts.sum()) == n
        graph.replay()
        torch.cuda.synchronize()
        assert int(plan.counts.sum()) == T * k
