"""DPGatedRNN, GroupNormAct and HeadNormAct on the CPU: construction, names, refusals, hook wiring."""

import copy

import pytest
import torch
import torch.nn as nn

from opacus_amd import GradSampleModule, GradSampleModuleFastGradientClipping
from opacus_amd.layers import DPGatedRNN, GatedScan, GroupNormAct, HeadNormAct


def test_construction_and_refusals():
    m = DPGatedRNN(6, 8, num_layers=2, bidirectional=True, num_heads=4)
    assert len(m.cells) == 4 and m.cells[2].ih.in_features == 16 and m.cells[1].scan.reverse
    half = torch.exp(-0.5 * nn.functional.softplus(m.cells[0].scan.decay))
    assert (half > 0.8999).all() and (half < 0.9991).all()
    assert m.initial_state(3).shape == (2, 3, 8)
    other = DPGatedRNN(6, 8, num_layers=2, bidirectional=True, num_heads=4)
    other.load_state_dict(m.state_dict())
    for bad in (dict(num_layers=0), dict(dropout=1.5), dict(num_heads=3), dict(num_heads=0)):
        with pytest.raises(ValueError):
            DPGatedRNN(6, 8, **bad)
    with pytest.raises(ValueError, match="bidirectional"):
        m.step(torch.zeros(3, 6), m.initial_state(3))
    one = DPGatedRNN(6, 8)
    with pytest.raises(ValueError, match="one token"):
        one.step(torch.zeros(3, 1, 6), one.initial_state(3))
    with pytest.raises(ValueError, match="state must be"):
        one.step(torch.zeros(3, 6), one.initial_state(2))
    with pytest.raises(ValueError, match="batch of sequences"):
        one(torch.zeros(3, 6))
    with pytest.raises(ValueError, match="state_init"):
        one(torch.zeros(5, 3, 6), torch.zeros(1, 2, 8))
    with pytest.raises(ValueError, match="own lengths"):
        one(nn.utils.rnn.pack_sequence([torch.zeros(2, 6)]), lengths=torch.tensor([2]))
    with pytest.raises(ValueError, match="reverse"):
        GatedScan(4, reverse=True).step(torch.zeros(1, 12), torch.zeros(1, 4))
    for cls in (GroupNormAct, HeadNormAct):
        with pytest.raises(ValueError, match="divisible"):
            cls(3, 8)
        with pytest.raises(ValueError, match="activation"):
            cls(2, 8, activation="tanh")
        with pytest.raises(ValueError, match="channels"):
            cls(2, 8)(torch.zeros(2, 5))
        assert cls(2, 8, affine=False).weight is None
    with pytest.raises(RuntimeError, match="GPU only"):
        one(torch.zeros(5, 3, 6))


@pytest.mark.parametrize("cls", [GradSampleModule, GradSampleModuleFastGradientClipping])
def test_functorch_is_refused_and_leaves_the_model_usable(cls):
    m = DPGatedRNN(4, 4, num_heads=2)
    with pytest.raises(NotImplementedError, match="functorch"):
        cls(m, force_functorch=True)

    class Owner(nn.Module):  # a layer without a sampler: its whole subtree would be differentiated functionally
        def __init__(self):
            super().__init__()
            self.scale, self.norm = nn.Parameter(torch.ones(4)), HeadNormAct(2, 4)

    with pytest.raises(NotImplementedError, match="HeadNormAct"):
        cls(Owner())
    cls(m)


def test_rows_are_kept_for_hooked_modules_only():
    from opacus_amd.layers.param_rows import parameter_rows

    scan = GatedScan(4)
    rows = parameter_rows(scan, (scan.decay,), 3)
    assert rows.shape == (3, 4) and "_dpk_param_rows" not in scan.__dict__
    wrapped = GradSampleModule(scan)
    parameter_rows(scan, (scan.decay,), 3)
    assert "_dpk_param_rows" in scan.__dict__
    wrapped.remove_hooks()
    assert "_dpk_param_rows" not in scan.__dict__ and "_dpk_rows_hooked" not in scan.__dict__
    norm = HeadNormAct(2, 4)
    rows = parameter_rows(norm, (norm.weight, norm.bias), 0)
    assert rows.shape == (0, 2, 4)
    rows.sum().backward()
    assert (norm.weight.grad == 0).all()


@pytest.mark.parametrize("make", [lambda: GatedScan(4), lambda: HeadNormAct(2, 12), lambda: GroupNormAct(3, 12)])
@pytest.mark.parametrize("cls", [GradSampleModule, GradSampleModuleFastGradientClipping])
def test_a_refused_call_leaves_nothing_on_the_module(cls, make):
    """A wrapped model whose forward pass raised (here: CPU tensors) can still be copied and used."""
    module = make()
    wrapped = cls(module)
    with pytest.raises(RuntimeError, match="GPU only"):
        wrapped(torch.zeros(2, 12, 12))
    assert "_dpk_param_rows" not in module.__dict__ and not getattr(module, "activations", [])
    other = copy.deepcopy(module)
    assert all(torch.equal(p, q) for p, q in zip(module.parameters(), other.parameters()))
