"""A mixture that has been called can be copied, saved and loaded: the plan of its last call stays behind."""
import copy
import io

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_copies_and_saved_modules():
    from mace_onegpu.expert_mix import ExpertMix
    m = ExpertMix(channels=32, n_experts=4, k=2)
    h = torch.randn(50, 4, 32, generator=torch.Generator().manual_seed(1)).cuda()
    want = m(h)
    m.update_balance()
    other = copy.deepcopy(m)
    assert other.plan is None and m.plan is not None
    file = io.BytesIO()
    torch.save(m, file)
    file.seek(0)
    loaded = torch.load(file, weights_only=False)      # written by this test
    m.balance.zero_()
    assert torch.equal(m(h), want)
    for n in (other, loaded):
        assert torch.equal(n.balance.abs(), torch.full((4,), 1e-2, device="cuda") * (n.balance != 0))
        n.balance.zero_()
        assert torch.equal(n(h), want)
