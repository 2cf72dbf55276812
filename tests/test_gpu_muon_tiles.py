"""orthogonalize by tiles of 64, 128 and 256, with the long side in parts, and in several parts of the batch: against the
iteration in 64 bits, and a matrix's bits whatever stands beside it (batches choose their tiles by how many there are).

The tolerance is that of test_gpu_muon.py, with bounds for its spectral norms: |X| <= 1 at first, and the largest value of
the step's polynomial over what was before."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
C = (3.4445, -4.7750, 2.0315)


def _matrices(E, m, n, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = max(1, min(m, n) // 8)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    strong = torch.bmm(rand(E, m, r) * torch.exp(rand(E, 1, r)), rand(E, r, n)) / r ** 0.5
    return (0.01 * (strong + 0.3 * rand(E, m, n))).to(dtype)


def _reference(m, dtype, steps=5, eps=1e-7):
    x = m.double()
    tall = x.shape[0] > x.shape[1]
    x = x.T.contiguous() if tall else x
    x = x / (torch.linalg.matrix_norm(x) + eps)
    fro = lambda t: float(torch.linalg.matrix_norm(t))  # noqa: E731
    r = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22
    n = max(x.shape)
    err = 4 * U * fro(x)
    a, b, c = C
    s = 1.0
    for _ in range(steps):
        A = x @ x.T.contiguous()
        B = b * A + c * A @ A
        t = torch.linspace(0, s, 1000, dtype=torch.float64)
        f, sA, sB = fro(x), s * s, float((b * t ** 2 + c * t ** 4).abs().max())
        dA = 2 * r * s * f + r * fro(A) + 3 * n * U * fro(x.abs() @ x.abs().T.contiguous())
        dB = (r * fro(B) + (abs(b) + 2 * abs(c) * sA) * dA
              + abs(c) * (2 * r * sA * fro(A) + 3 * n * U * fro(A.abs() @ A.abs())))
        new = a * x + B @ x
        noise = 2 * r * sB * f + s * dB + 3 * n * U * fro(B.abs() @ x.abs()) + 4 * U * (a * f + fro(new))
        gain = max(abs(a), float((a + 3 * b * t ** 2 + 5 * c * t ** 4).abs().max()))
        err = gain * err + noise
        x, s = new, float((a * t + b * t ** 3 + c * t ** 5).abs().max())
    out = x.T if tall else x
    return out, err + HALF_ULP[dtype] * fro(out)


# Tiles of the squares and of the steps (bfloat16; float32 and float16): 64, 128; 256, 128 and 128, 256 (two parts of the
# batch); 128, 256 and 64, 128; 128, 256; 64, 128 in two parts; 256, 256 and 128, 128 in two parts.  Single ones: 64.
SIZES = [(24, 500, 515), (60, 500, 515), (60, 515, 500), (8, 1100, 1300), (9, 1000, 1000), (150, 300, 705),
         (150, 705, 300), (230, 250, 250)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,m,n", SIZES)
def test_batches_by_tiles(E, m, n, dtype):
    from mace_onegpu.muon import orthogonalize
    M = _matrices(E, m, n, dtype, E + m + n)
    got = orthogonalize(M)
    assert torch.equal(got, orthogonalize(M))
    for e in sorted({0, E // 2, E - 1}):
        want, bound = _reference(M[e], dtype)
        err = float(torch.linalg.matrix_norm(got[e].double() - want))
        assert err <= bound, (e, err, bound)
    for e in range(0, E, 7):
        assert torch.equal(got[e], orthogonalize(M[e])), e
    some = list(range(E - 1, -1, -3))
    assert torch.equal(got[some], orthogonalize(M[some]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,m,n", [(1, 2100, 2300), (1, 4500, 4400)])
def test_large_matrices(E, m, n, dtype):
    from mace_onegpu.muon import orthogonalize
    M = _matrices(E, m, n, dtype, m)
    want, bound = _reference(M[0], dtype)
    err = float(torch.linalg.matrix_norm(orthogonalize(M)[0].double() - want))
    assert err <= bound, (err, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,m,n", [(1, 100, 1500), (3, 1025, 192), (2, 192, 4100), (2, 5000, 70), (1, 3, 9000)])
def test_long_sides_in_parts(E, m, n, dtype):
    from mace_onegpu.muon import orthogonalize
    M = _matrices(E, m, n, dtype, m + n)
    got = orthogonalize(M)
    for e in range(E):
        want, bound = _reference(M[e], dtype)
        err = float(torch.linalg.matrix_norm(got[e].double() - want))
        assert err <= bound, (e, err, bound)
        assert torch.equal(got[e], orthogonalize(M[e]))
