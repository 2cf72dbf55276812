"""Group norm, linear cross entropy and orthogonalisation called by several host threads at once, each on its own stream;
weights that are their own rows."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_threads():
    from mace_onegpu.cross_entropy import linear_cross_entropy
    from mace_onegpu.group_norm import group_norm
    from mace_onegpu.muon import orthogonalize
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    y, o = torch.randint(0, 3000, (200,), generator=g).cuda(), torch.tensor([0, 3, 150, 150, 2000]).cuda()

    def loss(x, w):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        value = linear_cross_entropy(x, w, y)
        return (value.detach(), *torch.autograd.grad(value, (x, w)))

    def norm(x):
        x = x.detach().requires_grad_()
        z = group_norm(x, 8, activation="gelu", offsets=o)
        return z.detach(), *torch.autograd.grad(z, x, x.detach())

    jobs = [(loss, (r(200, 128), r(3000, 128))), (norm, (r(2010, 64),)), (lambda m: (orthogonalize(m),), (r(3, 200, 300),)),
            (lambda m: (orthogonalize(m),), (r(9, 100, 60).bfloat16(),))]
    want = [f(*a) for f, a in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        f, args = jobs[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = f(*args)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_rows_of_the_weight_as_input():
    """x is a part of weight: its gradient is the sum of both."""
    from mace_onegpu.cross_entropy import linear_cross_entropy
    g = torch.Generator().manual_seed(1)
    w = (torch.randn(90, 48, generator=g) / 7).cuda().requires_grad_()
    y = torch.randint(0, 90, (30,), generator=g).cuda()
    for rows in (slice(0, 30), slice(0, 90, 3), slice(5, 6)):
        n = len(range(90)[rows])
        got, = torch.autograd.grad(linear_cross_entropy(w[rows], w, y[:n]), w)
        x = w.detach()[rows].clone().requires_grad_()
        dx, dw = torch.autograd.grad(linear_cross_entropy(x, w, y[:n]), (x, w))
        dw[rows] += dx
        assert torch.equal(got, dw)
