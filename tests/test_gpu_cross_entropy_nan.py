"""A NaN logit reaches the loss wherever its class stands, in few rows as in many.  Classes are taken four a wave: 0 and 4
are the first that a wave meets, 5 is not, 0 .. 5 a run of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [[0], [4], [5], list(range(6)), [48]])
@pytest.mark.parametrize("V", [49, 3001])        # one workgroup, several
@pytest.mark.parametrize("T", [1, 5, 16, 17])
def test_nan_weight_row(T, V, bad, dtype):
    from mace_onegpu.cross_entropy import linear_cross_entropy
    g = torch.Generator().manual_seed(T + V)
    x = torch.randn(T, 64, generator=g).to(dtype).cuda().requires_grad_()
    w = torch.randn(V, 64, generator=g).to(dtype)
    w[bad] = float("nan")
    y = torch.full((T,), 7).cuda()
    loss = linear_cross_entropy(x, w.cuda(), y, reduction="none")
    assert loss.isnan().all()
    assert linear_cross_entropy(x, w.cuda(), y).isnan()
    dx, = torch.autograd.grad(loss.sum(), x)
    assert dx.isnan().all()
