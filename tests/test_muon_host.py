"""Muon's parameter groups and saved state (no GPU: nothing is stepped)."""
import pytest
import torch


def test_a_refused_group_is_not_kept():
    from mace_onegpu.muon import Muon
    good, vector = torch.nn.Parameter(torch.zeros(3, 4)), torch.nn.Parameter(torch.zeros(4))
    opt = Muon([good])
    for group in (dict(params=[vector]), dict(params=vector),
                  dict(params=[torch.nn.Parameter(torch.zeros(2, 2)), vector])):
        with pytest.raises(ValueError, match="matrices"):
            opt.add_param_group(group)
        assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2, 3, 4))], lr=0.5))
    assert [g["lr"] for g in opt.param_groups] == [1e-3, 0.5]


def test_state_of_parameters_that_had_no_gradient():
    """An empty entry, which looking at opt.state[p] makes, is saved and loaded like none."""
    from mace_onegpu.muon import Muon
    p = [torch.nn.Parameter(torch.zeros(3, 4, dtype=torch.bfloat16)) for _ in range(3)]
    opt = Muon(p)
    assert "momentum_buffer" not in opt.state[p[0]]
    opt.state[p[2]]["momentum_buffer"] = torch.full((3, 4), 1.001)
    saved = opt.state_dict()
    new = Muon(p)
    new.load_state_dict(saved)
    assert not new.state[p[0]] and not new.state[p[1]]
    buf = new.state[p[2]]["momentum_buffer"]
    assert buf.dtype == torch.float32 and torch.equal(buf, torch.full((3, 4), 1.001))
    assert buf.data_ptr() != opt.state[p[2]]["momentum_buffer"].data_ptr()
