"""Infinities and NaN in the products' operands: where they may show, where they must not, and the same for a row alone as
among many rows.  All comparisons are exact (bits, or classes of values)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")
ROUNDS_TO_INF = (2 - 2.0 ** -8) * 2.0 ** 127      # the least float32 whose bfloat16 is infinity: 3.396e38
BELOW = (2 - 2.0 ** -8 - 2.0 ** -23) * 2.0 ** 127
# few rows; one choice (held / tiles); pairs (held / tiles of 16 bits); slots
CASES = [(7, 64, 48, 4, 2), (600, 64, 64, 4, 1), (600, 200, 136, 4, 1), (40000, 64, 64, 3, 2), (140000, 64, 128, 3, 2),
         (2000, 72, 56, 8, 3)]


def _case(T, D, F, E, k, dtype):
    g = torch.Generator().manual_seed(T + D)
    x, w = torch.randn(T, D, generator=g).to(dtype).cuda(), torch.randn(E, D, F, generator=g).to(dtype).cuda()
    e = torch.rand(T, E, generator=g).topk(k, 1).indices.to(torch.int32).cuda()
    dy = torch.randn(T, F, generator=g).to(dtype).cuda()
    return x, w, e, torch.rand(T, k, generator=g).cuda() + 0.5, dy


def _all(x, w, e, gates, dy):
    from mace_onegpu.experts import expert_linear, plan_experts
    a, b, c = (t.clone().requires_grad_() for t in (x, w, gates))
    y = expert_linear(a, b, plan_experts(e, w.shape[0]), c)
    return (y.detach(),) + torch.autograd.grad(y, (a, b, c), dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,F,E,k", CASES)
def test_closed_slots_hide_everything(T, D, F, E, k, dtype):
    """Whatever stands in rows without an expert and in the gates of closed slots: no other value changes, theirs are 0."""
    x, w, e, gates, dy = _case(T, D, F, E, k, dtype)
    closed = torch.arange(T, device="cuda") % 5 == 2
    e[closed] = -1
    e[1, 0] = E                                                       # half a row, unless there is one choice
    want = _all(x, w, e, gates, dy)
    x[closed], dy[closed], gates[closed] = INF, float("nan"), float("nan")
    gates[1, 0] = float("nan")
    got = _all(x, w, e, gates, dy)
    for p, q in zip(want, got):
        assert torch.equal(p, q)
    assert not got[0][closed].any() and not got[1][closed].any() and not got[3][closed].any() and not got[3][1, 0]


@pytest.mark.parametrize("value", [INF, -INF, float("nan"), ROUNDS_TO_INF, -ROUNDS_TO_INF])
@pytest.mark.parametrize("T,D,F,E,k", CASES)
def test_float_rows_and_blocks(T, D, F, E, k, value):
    """float32: what rounds to infinity in bfloat16 gives NaN, in its row or column and nowhere else."""
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, e, gates, _ = _case(T, D, F, E, k, torch.float32)
    plan = plan_experts(e, E)
    want = expert_linear(x, w, plan, gates)
    x[3, 5] = value
    y = expert_linear(x, w, plan, gates)
    assert bool(y[3].isnan().all()) and torch.equal(y[:3], want[:3]) and torch.equal(y[4:], want[4:])
    x[3, 5] = 0.0
    want = expert_linear(x, w, plan, gates)
    w[1, 7, 9] = value
    y = expert_linear(x, w, plan, gates)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[(e == 1).any(1), 9] = True
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], want[~bad])


@pytest.mark.parametrize("T,D,F,E,k", CASES)
def test_largest_floats_are_finite(T, D, F, E, k):
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, e, gates, _ = _case(T, D, F, E, k, torch.float32)
    x[3], w[:, 5] = 0.0, 2.0 ** -100
    x[3, 5] = BELOW
    y = expert_linear(x, w, plan_experts(e, E), gates)[3].double()
    want = gates[3].double().sum() * BELOW * 2.0 ** -100
    assert float((y / want - 1).abs().max()) < 1e-5      # one product and a gate a choice: a few units of 2^-24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D,F,E,k", CASES)
def test_16_bit_rows_follow_the_sums(T, D, F, E, k, dtype):
    """16-bit types multiply as they are: infinity or NaN exactly as in 64-bit sums, on every path."""
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, e, gates, _ = _case(T, D, F, E, k, dtype)
    x[0, 5], x[2, 0], x[2, 1], x[3, 4], w[1, 7, 9], w[1, 8, 10], w[0, 3, 3] = INF, INF, -INF, float("nan"), INF, -INF, 0.0
    y = expert_linear(x, w, plan_experts(e, E), gates)
    rows = torch.arange(min(T, 600), device="cuda")
    xd, wd = x[rows].double(), w.double()
    ref = sum(gates[rows, j, None].double() * (xd[:, :, None] * wd[e[rows, j].long()]).sum(1) for j in range(k))
    got = y[rows].double()
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.isinf(), ref.isinf())
    assert torch.equal(got[ref.isinf()], ref[ref.isinf()])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,F,E,k", CASES)
def test_a_row_alone_is_as_among_many(T, D, F, E, k, dtype):
    from mace_onegpu.experts import expert_linear, plan_experts
    x, w, e, gates, _ = _case(T, D, F, E, k, dtype)
    x[0, 5], x[1, 0], x[2, 3], x[2, 4] = INF, -INF, INF, float("nan")
    w[1, 7, 9] = INF
    y = expert_linear(x, w, plan_experts(e, E), gates)
    for t in range(4):
        one = expert_linear(x[t:t + 1], w, plan_experts(e[t:t + 1], E), gates[t:t + 1])
        for f in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(f(one[0]), f(y[t]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,F,E,k", CASES)
def test_gradients_keep_them_in_their_places(T, D, F, E, k, dtype):
    """An infinite value of x or of the cotangent: not finite in the gradients that it enters, all others unchanged."""
    x, w, e, gates, dy = _case(T, D, F, E, k, dtype)
    _, dx, dw, dg = _all(x, w, e, gates, dy)
    of_3 = torch.zeros(E, dtype=torch.bool, device="cuda")
    of_3[e[3].long()] = True
    x[3, 5] = INF
    _, bx, bw, bg = _all(x, w, e, gates, dy)
    assert torch.equal(bx, dx) and torch.equal(bg[:3], dg[:3]) and torch.equal(bg[4:], dg[4:])
    assert not bg[3].isfinite().any() and not bw[of_3][:, 5].isfinite().any()
    bw[of_3, 5] = dw[of_3, 5] = 0
    assert torch.equal(bw, dw)
    x[3, 5] = 1.0
    _, dx, dw, dg = _all(x, w, e, gates, dy)
    dy[3, 6] = -INF
    _, bx, bw, bg = _all(x, w, e, gates, dy)
    for b, d in ((bx, dx), (bg, dg)):
        assert not b[3].isfinite().any() and torch.equal(b[:3], d[:3]) and torch.equal(b[4:], d[4:])
    assert not bw[of_3][:, :, 6].isfinite().any()
    bw[of_3, :, 6] = dw[of_3, :, 6] = 0
    assert torch.equal(bw, dw)
