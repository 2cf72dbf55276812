"""dW of 16-bit types with gates, against 64 bits: gate x dy is not rounded to the type on the way.

Tolerance, element by element, from the formats: gate x dy in float32 (u = 2^-24) is two bfloat16 parts, off by 2^-18 of
it; float16 rows are two bfloat16 parts exactly, and the product of the two second parts (2^-18) is left out: 2^-17 of
the sum of magnitudes in all.  A float32 sum of n products: (n + 16) u of it.  Rounding to the output's type adds half a
unit in its last place: 2^-8 (bfloat16), 2^-11 (float16) of the result, for float16 at least half its least value.
Ranges that the products gate x dy leave are part of it: float16 has no 1e-8 and nothing above 65504."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}


def _dw(x, w_shape, experts, gates, dy):
    from mace_onegpu.experts import expert_linear, plan_experts
    w = torch.zeros(w_shape, dtype=x.dtype, device="cuda", requires_grad=True)
    y = expert_linear(x.cuda(), w, plan_experts(experts.cuda(), w_shape[0]), None if gates is None else gates.cuda())
    (dw,) = torch.autograd.grad(y, w, dy.cuda())
    return dw


def _check(T, M, D, F, E, k, dtype, seed, dy_size, gate_size, x_size=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (x_size * torch.randn(T, M, D, generator=g)).to(dtype)
    dy = (dy_size * torch.randn(T, M, F, generator=g)).to(dtype)
    experts = torch.rand(T, E, generator=g).topk(k, 1).indices.to(torch.int32)
    experts[torch.rand(T, k, generator=g) < 0.05] = -1
    gates = gate_size * torch.rand(T, k, generator=g) if gate_size else None
    ref, mag = torch.zeros(E, D, F, dtype=torch.float64), torch.zeros(E, D, F, dtype=torch.float64)
    rows = 0
    for e in range(E):
        t, j = (experts == e).nonzero(as_tuple=True)
        a = dy[t].double() if gates is None else gates[t, j].double()[:, None, None] * dy[t].double()
        a = a.reshape(-1, F)
        b = x[t].double().reshape(-1, D)
        ref[e], mag[e] = b.T @ a, b.abs().T @ a.abs()
        rows = max(rows, t.numel() * M)
    bound = (2.0 ** -17 + (rows + 16) * U) * mag + HALF_ULP[dtype] * ref.abs() + TINY[dtype]
    dw = _dw(x, (E, D, F), experts, gates, dy)
    # cotangents of 15000 now and then pass float16's largest value: their columns, and no others, are not finite
    finite = ref.isfinite()
    assert dw.dtype == dtype and torch.equal(dw.isfinite().cpu(), finite)
    err, bound = (dw.double().cpu() - ref).abs()[finite], bound[finite]
    assert bool((err <= bound).all()), (float((err - bound).max()), float((err / bound).max()))


# tiles of 64 and 128, chunks and whole lists, the 256 x 256 tiles (16 experts of 1536 x 1536), odd widths, components
SIZES = [(700, 1, 128, 128, 8, 2), (300, 3, 72, 56, 5, 2), (4001, 1, 201, 137, 9, 3), (900, 2, 40, 130, 4, 1),
         (600, 1, 136, 48, 3, 2), (60, 1, 33, 47, 3, 2), (1200, 1, 1536, 1536, 16, 2), (2000, 1, 640, 512, 32, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,M,D,F,E,k", SIZES)
def test_gates_are_not_rounded(T, M, D, F, E, k, dtype):
    _check(T, M, D, F, E, k, dtype, T + D, 1.0, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dy_size,gate_size,x_size", [(1e-5, 1e-2, 100.0), (1e-6, 0.1, 1000.0), (1e-4, 0.1, 30.0),
                                                      (15000.0, 8.0, 1e-4), (8000.0, 2.5, 1e-3)])
@pytest.mark.parametrize("T,M,D,F,E,k", [(700, 1, 128, 128, 8, 2), (4001, 1, 201, 137, 9, 3)])
def test_small_and_large_cotangents(T, M, D, F, E, k, dy_size, gate_size, x_size, dtype):
    """Cotangents whose product with a gate is below float16's least value or above its largest, and a dW in range."""
    _check(T, M, D, F, E, k, dtype, T + D + 1, dy_size, gate_size, x_size)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,M,D,F,E,k", SIZES)
def test_without_gates(T, M, D, F, E, k, dtype):
    _check(T, M, D, F, E, k, dtype, T + D + 2, 1.0, None)
