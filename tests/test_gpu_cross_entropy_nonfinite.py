"""float32 values that round to infinity in bfloat16 (from 3.396e38 on, infinity among them) give NaN in the losses that
they enter, for one row as for many, whatever they are multiplied with; 16-bit infinities give what their sums do."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(T, V, dtype):
    g = torch.Generator().manual_seed(T + V)
    x, w = torch.randn(T, 40, generator=g), torch.randn(V, 40, generator=g)
    x[:, 3] = 0.0
    w[:, 5] = 0.0
    return x.to(dtype).cuda(), w.to(dtype).cuda(), torch.full((T,), 2).cuda()


@pytest.mark.parametrize("value", [3.3961776e38, torch.finfo(torch.float32).max, -3.4e38, float("inf"), -float("inf")])
@pytest.mark.parametrize("V", [30, 2000])
@pytest.mark.parametrize("T", [1, 4, 16, 17, 70])
def test_large_floats(T, V, value):
    from mace_onegpu.cross_entropy import linear_cross_entropy as f
    x, w, y = _inputs(T, V, torch.float32)
    plain = f(x, w, y, reduction="none")
    assert plain.isfinite().all()
    for v in (V - 1, 0, 9):                        # met by zeros of x: the logit of one class
        bad = w.clone()
        bad[v, 3] = value
        assert f(x, bad, y, reduction="none").isnan().all()
    bad = x.clone()
    bad[T // 2, 5] = value                         # met by zeros of w: all logits of one row
    loss = f(bad, w, y, reduction="none")
    assert bool(loss[T // 2].isnan())
    loss[T // 2] = plain[T // 2]
    assert torch.equal(loss, plain)


@pytest.mark.parametrize("T", [1, 4, 16, 17, 70])
def test_floats_below_the_limit(T):
    from mace_onegpu.cross_entropy import linear_cross_entropy as f
    x, w, y = _inputs(T, 30, torch.float32)
    plain = f(x, w, y, reduction="none")
    w[5, 3] = 3.396e38
    x[0, 5] = -3.396e38
    assert torch.equal(f(x, w, y, reduction="none"), plain)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 4, 16, 17, 70])
def test_infinite_half_weights(T, dtype):
    """A class whose logit is minus infinity has probability 0; plus infinity, or NaN, gives NaN."""
    from mace_onegpu.cross_entropy import linear_cross_entropy as f
    x, w, y = _inputs(T, 30, dtype)
    x[:, 3] = 1.0
    cut = w.clone()
    cut[9, 3] = -float("inf")
    without = torch.cat([w[:9], w[10:]])
    got, want = f(x, cut, y, reduction="none"), f(x, without, y, reduction="none")
    assert float((got - want).abs().max()) <= 2.0 ** -20 * float(want.abs().max() + 8)
    cut[9, 3] = float("inf")
    assert f(x, cut, y, reduction="none").isnan().all()
