"""group_norm of many ragged structures of which a few are long: one wave a structure together with tiles, the joins by
one wave (256 structures and more), and with fewer by a workgroup; against the formula in 64 bits, with the tolerances of
test_gpu_group_norm.py."""
import pytest
import torch

from test_gpu_group_norm import _check, _inputs, _reference, _run

pytestmark = pytest.mark.gpu


def _bounds(structs, seed, first):
    """Structures of 0 - 30 rows; every 40th of 200 - 1000, one of which begins on a multiple of 256 rows (a border of
    its tiles, whatever power of two up to it they have), the next of which begin inside one."""
    g = torch.Generator().manual_seed(seed)
    sizes = torch.randint(0, 31, (structs,), generator=g)
    sizes[::5] = 0
    long = torch.arange(7, structs, 40)
    sizes[long] = torch.randint(200, 1001, (long.numel(),), generator=g)
    sizes[6] += -(first + int(sizes[:7].sum())) % 256
    return [first] + (first + torch.cumsum(sizes, 0)).tolist()


@pytest.mark.parametrize("dtype,C,G,kind", [(torch.float32, 128, 8, "silu"), (torch.bfloat16, 128, 8, "gelu"),
                                            (torch.float16, 64, 4, "silu"), (torch.float32, 24, 3, "gelu"),
                                            (torch.bfloat16, 70, 2, "none"), (torch.float32, 256, 1, "none")])
@pytest.mark.parametrize("structs", [200, 300, 3000])
def test_few_long_structures_among_many(structs, dtype, C, G, kind):
    bounds = _bounds(structs, structs + C, 5)
    rows = bounds[-1] + 17
    x, w, b, dy = _inputs(rows, C, dtype, dtype, structs + C)
    ref, bound = _reference(x, w, b, dy, bounds, G, 1e-5, kind, dtype, dtype)
    got = _run(x, w, b, dy, G, kind, torch.tensor(bounds, dtype=torch.int32).cuda())
    _check(got, ref, bound)
    again = _run(x, w, b, dy, G, kind, torch.tensor(bounds).cuda())
    assert all(torch.equal(got[n], again[n]) for n in got)
    for t in (got["y"], got["dx"]):
        assert not t[:bounds[0]].any() and not t[bounds[-1]:].any()
