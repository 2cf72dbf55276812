"""Muon's first step makes its momentum.  Made inside a graph it would be cleared by every replay, so a captured step is
refused until there is one; after an eager step, replays carry the momentum on."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_first_step_in_a_capture_is_refused():
    from mace_onegpu.muon import Muon
    g = torch.Generator().manual_seed(0)
    p, q = (torch.nn.Parameter(torch.zeros(3, 24, 40, device="cuda")) for _ in range(2))
    grads = [torch.randn(3, 24, 40, generator=g).cuda() for _ in range(5)]
    p.grad, q.grad = grads[0].clone(), grads[0].clone()
    opt, eager = Muon([p], lr=0.01), Muon([q], lr=0.01)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before it is captured"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert not p.detach().any() and not opt.state[p]
    opt.step()
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for t in grads[1:]:
        p.grad.copy_(t)
        q.grad.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        eager.step()
        assert torch.equal(p.detach(), q.detach())
        assert torch.equal(opt.state[p]["momentum_buffer"], eager.state[q]["momentum_buffer"])
