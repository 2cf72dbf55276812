"""Captures that use a plan whose lists were sorted before: on the default stream, on the capture's own stream, and on a
stream that takes part in the capture."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CASES = [(20000, 1, 6, torch.float32), (40000, 2, 3, torch.float32), (30000, 3, 8, torch.float16)]


def _case(T, k, E, dtype):
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, 64, generator=g).to(dtype).cuda()
    w = torch.randn(E, 64, 64, generator=g).to(dtype).cuda()
    e = torch.rand(T, E, generator=g).topk(k, 1).indices.to(torch.int32).cuda()
    return x, w, e, torch.rand(T, k, generator=g).cuda()


def _replays(graph, x, ys, want):
    for scale in (2.0, 0.5, 1.0):
        x.mul_(scale)
        graph.replay()
        torch.cuda.synchronize()
        for y in ys:
            assert torch.equal(y, want())


@pytest.mark.parametrize("T,k,E,dtype", CASES)
def test_lists_of_the_default_stream(T, k, E, dtype):
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, e, gates = _case(T, k, E, dtype)
    plan = plan_experts(e, E)
    assert torch.cuda.current_stream() == torch.cuda.default_stream()
    expert_linear(x, w, plan, gates)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = expert_linear(x, w, plan, gates)
    _replays(graph, x, [y], lambda: expert_linear(x, w, plan, gates))


@pytest.mark.parametrize("T,k,E,dtype", CASES)
def test_lists_of_the_capturing_streams(T, k, E, dtype):
    """The capture forks to the stream that sorted the lists, and uses them on both."""
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, e, gates = _case(T, k, E, dtype)
    for first in (0, 1):
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        plan = plan_experts(e, E)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[first]):
            expert_linear(x, w, plan, gates)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            streams[1].wait_stream(streams[0])
            y = expert_linear(x, w, plan, gates)
            with torch.cuda.stream(streams[1]):
                z = expert_linear(x, w, plan, gates)
            streams[0].wait_stream(streams[1])
        _replays(graph, x, [y, z], lambda: expert_linear(x, w, plan_experts(e, E), gates))
