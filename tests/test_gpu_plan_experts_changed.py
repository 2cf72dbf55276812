"""A plan reads the caller's int32 experts again at every product: changed in place, they are refused, not mixed with
lists of the old ones.  Copies (int64, strided) are the plan's own."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CASES = [(40, 2, 8), (20000, 2, 3), (5000, 3, 8), (3000, 1, 5)]      # few rows, pairs, slots, one choice


def _case(T, k, E):
    g = torch.Generator().manual_seed(T)
    x, w = torch.randn(T, 64, generator=g).cuda(), torch.randn(E, 64, 48, generator=g).cuda()
    e = [torch.rand(T, E, generator=g).topk(k, 1).indices.to(torch.int32).cuda() for _ in range(2)]
    return x, w, torch.rand(T, k, generator=g).cuda(), e


@pytest.mark.parametrize("use_first", [False, True])
@pytest.mark.parametrize("T,k,E", CASES)
def test_changed_experts_are_refused(T, k, E, use_first):
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, gates, (old, new) = _case(T, k, E)
    want = expert_linear(x, w, plan_experts(new.clone(), E), gates)
    experts = old.clone()
    plan = plan_experts(experts, E)
    if use_first:
        expert_linear(x, w, plan, gates)
        plan.counts
    experts.copy_(new)
    for call in (lambda: expert_linear(x, w, plan, gates), lambda: plan.counts, lambda: plan.order,
                 lambda: expert_linear(x.clone().requires_grad_(), w, plan, gates)):
        with pytest.raises(RuntimeError, match="changed in place"):
            call()
    assert torch.equal(expert_linear(x, w, plan_experts(experts, E), gates), want)     # a new plan of the same buffer


@pytest.mark.parametrize("T,k,E", CASES)
def test_copies_are_the_plans_own(T, k, E):
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, gates, (old, new) = _case(T, k, E)
    want = expert_linear(x, w, plan_experts(old, E), gates)
    wide = torch.zeros(T, k + 1, dtype=torch.int32, device="cuda")
    for experts in (old.long(), wide[:, 1:]):
        experts.copy_(old)
        plan = plan_experts(experts, E)
        experts.copy_(new)
        assert torch.equal(expert_linear(x, w, plan, gates), want)
        assert torch.equal(plan.counts.long(), torch.bincount(old.reshape(-1).long(), minlength=E))


@pytest.mark.parametrize("T,k,E", CASES)
def test_inference_mode(T, k, E):
    from mace_onegpu.experts import expert_linear, plan_experts, route
    x, w, gates, (old, _) = _case(T, k, E)
    want = expert_linear(x, w, plan_experts(old, E), gates)
    with torch.inference_mode():
        plan = plan_experts(old.clone(), E)
        assert torch.equal(expert_linear(x, w, plan, gates), want) and int(plan.counts.sum()) == T * k
        g, e = route(torch.randn(T, E, generator=torch.Generator().manual_seed(1)).cuda(), k)
        assert expert_linear(x, w, plan_experts(e, E), g).shape == want.shape


def test_a_buffer_written_between_replays():
    """Inside a graph the experts' buffer may change from replay to replay."""
    from mace_onegpu.experts import expert_linear, plan_experts
    for T, k, E in CASES:
        x, w, gates, both = _case(T, k, E)
        experts = both[0].clone()
        expert_linear(x, w, plan_experts(experts, E), gates)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan = plan_experts(experts, E)
            y = expert_linear(x, w, plan, gates)
        for e in (both[1], both[0], both[1]):
            experts.copy_(e)
            graph.replay()
            torch.cuda.synchronize()
            want = expert_linear(x, w, plan_experts(e, E), gates)
            assert torch.equal(y, want) and torch.equal(expert_linear(x, w, plan, gates), want)
