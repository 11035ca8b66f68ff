"""The Mamba-1 layer's calls that are refused before anything is launched (on the CPU)."""

import pytest
import torch

import mamba_hip


def layer():
    return mamba_hip.Mamba1Layer.init(mamba_hip.Mamba1Config(16), "cpu")


@pytest.mark.parametrize("which", ["norm_w", "norm_b", "d"])
@pytest.mark.parametrize("slots", [None, torch.zeros(2, dtype=torch.int32)])
def test_step_where_a_gradient_is_wanted(which, slots):
    m = layer()
    (m.mixer.d if which == "d" else getattr(m, which)).requires_grad_()
    with pytest.raises(mamba_hip.MambaHipError, match="differentiable"):
        m.step(torch.zeros(2, 16), m.mixer.new_cache(2), slots)


@pytest.mark.parametrize("trained", [False, True])
def test_slots_without_a_cache(trained):
    """With gradients too, where the call would start every sequence from zero."""
    m = layer().mixer
    m.d.requires_grad_(trained)
    with pytest.raises(mamba_hip.MambaHipError, match="slots without a cache"):
        m.forward_packed(torch.zeros(4, 16), torch.zeros(2, dtype=torch.int32), slots=torch.zeros(1, dtype=torch.int32))
