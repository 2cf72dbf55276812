"""What the balance bias is added to: the logits, whose order with a bias is not the order of score + bias, and a NaN's
reach.  Small rows by hand."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_bias_is_added_to_the_logits():
    from mace_onegpu.experts import route
    x = torch.tensor([[3.0, 1.0, -2.0, 0.0]], device="cuda")
    b = torch.tensor([0.0, 0.5, 4.5, 0.0], device="cuda")
    for scoring in ("sigmoid", "softmax"):
        gates, experts = route(x, 2, scoring=scoring, bias=b, renormalize=False)
        assert experts.tolist() == [[0, 2]]                      # keys 3, 1.5, 2.5, 0
        s = torch.sigmoid(x) if scoring == "sigmoid" else torch.softmax(x, 1)
        assert (s + b).topk(2, 1).indices.tolist() != experts.tolist()    # the other rule: scores + bias
        assert torch.allclose(gates, s[:, [0, 2]], rtol=1e-6)    # without the bias
        plain = route(x, 3, scoring=scoring)[1]
        assert plain.tolist() == s.topk(3, 1).indices.tolist()   # without a bias the orders agree


def test_groups_go_by_their_largest_key():
    from mace_onegpu.experts import route
    x = torch.tensor([[2.0, -5.0, 1.5, 1.4]], device="cuda")     # the second group has the larger sum of two
    assert route(x, 2, groups=2, top_groups=1)[1].tolist() == [[0, 1]]


def test_a_nan_logit():
    from mace_onegpu.experts import route
    x = torch.tensor([[0.5, 2.0, math.nan, 1.0], [0.5, 2.0, 3.0, 1.0]], device="cuda")
    for kw in (dict(), dict(renormalize=False), dict(scoring="sigmoid")):
        gates, experts = route(x, 2, **kw)
        assert experts.tolist() == [[2, 1], [2, 1]]
        assert bool(gates[0].isnan().all()) and bool(gates[1].isfinite().all())
    gates, experts = route(x, 2, scoring="sigmoid", renormalize=False)
    assert experts.tolist() == [[2, 1], [2, 1]] and gates.isnan().tolist() == [[True, False], [False, False]]
