"""Losses whose gradients are taken in several pieces of the classes with the products' sums in parts, against the formula
in 64 bits, with the tolerances of test_gpu_cross_entropy.py."""
import pytest
import torch

from test_gpu_cross_entropy import _check, _inputs, _reference, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,D,V,dtype", [(3001, 77, 32003, torch.float16), (3001, 40, 32003, torch.bfloat16),
                                         (3001, 40, 30000, torch.float32), (9000, 64, 9000, torch.bfloat16)])
def test_pieces_with_split_sums(T, D, V, dtype):
    x, w, y, dloss = (t.cuda() for t in _inputs(T, D, V, dtype, T + V))
    ref, bound = _reference(x, w, y, dloss, "none", dtype)
    got = _run(x, w, y, dloss, "none")
    _check(got, ref, bound)
    again = _run(x, w, y, dloss, "none")
    assert all(torch.equal(got[n], again[n]) for n in got)
