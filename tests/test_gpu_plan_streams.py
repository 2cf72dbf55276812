"""A plan shared by products on several streams that wait for the plan's stream only: every stream's result is that of a
fresh plan, whichever call sorted the lists, and the lists stay in memory until the last stream has read them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SLEEP = 20_000_000     # cycles that hold a stream back, some 10 ms


def _case(T, k, E, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, 1, 64, generator=g).to(dtype).cuda()
    w = torch.randn(E, 64, 64, generator=g).to(dtype).cuda()
    e = torch.rand(T, E, generator=g).topk(k, 1).indices.cuda()
    return x, w, e.to(torch.int32), torch.rand(T, k, generator=g).cuda()


# one choice; pairs (held, and in tiles for 16 bits); slots
CASES = [(20000, 1, 6, torch.float32), (40000, 2, 3, torch.float32), (280000, 2, 2, torch.bfloat16),
         (30000, 3, 8, torch.float16)]


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("T,k,E,dtype", CASES)
def test_two_streams(T, k, E, dtype, train):
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, e, gates = _case(T, k, E, dtype, T)
    dy = torch.randn(T, 1, 64, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()

    def product(plan):
        if not train:
            return (expert_linear(x, w, plan, gates),)
        a, b, c = (t.detach().requires_grad_() for t in (x, w, gates))
        y = expert_linear(a, b, plan, c)
        return (y,) + torch.autograd.grad(y, (a, b, c), dy)

    want = product(plan_experts(e, E))
    for experts in (e, e.long()):
        plan = plan_experts(experts, E)
        main, first, second = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()
        first.wait_stream(main)
        second.wait_stream(main)
        with torch.cuda.stream(first):
            torch.cuda._sleep(SLEEP)              # the lists come late
            got = product(plan)
        with torch.cuda.stream(second):
            again = product(plan)
            counts = plan.counts
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)) and all(torch.equal(a, b) for a, b in zip(want, again))
        assert torch.equal(counts.long(), torch.bincount(e.reshape(-1).long(), minlength=E))


@pytest.mark.parametrize("T,k,E,dtype", CASES)
def test_lists_outlive_their_plan(T, k, E, dtype):
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, e, gates = _case(T, k, E, dtype, T + 1)
    want = expert_linear(x, w, plan_experts(e, E), gates)
    plan = plan_experts(e.long(), E)              # an int32 copy that only the plan holds
    expert_linear(x, w, plan, gates)              # the lists are sorted on this stream
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        torch.cuda._sleep(SLEEP)
        y = expert_linear(x, w, plan, gates)
    del plan
    filler = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in range(T, 12 * T, T // 4)]
    torch.cuda.synchronize()
    assert torch.equal(y, want) and len(filler)


def test_capture_with_an_older_plan():
    """Lists sorted before the capture, on another stream, are taken as they are; unsorted ones are sorted in the graph."""
    from mace_onegpu.experts import expert_linear, plan_experts
    for T, k, E, dtype in CASES:
        x, w, e, gates = _case(T, k, E, dtype, T + 2)
        for sort_first in (True, False):
            plan = plan_experts(e, E)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                want = expert_linear(x, w, plan if sort_first else plan_experts(e, E), gates)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = expert_linear(x, w, plan, gates)
            for scale in (1.0, 2.0, 0.5):
                x.mul_(scale)
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(y, expert_linear(x, w, plan_experts(e, E), gates))
            assert torch.equal(y, want)           # x is as it was: 1 x 2 x 0.5
