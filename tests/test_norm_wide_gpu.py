"""Layer norm gradients of a row wider than a grid of one workgroup a 16 columns."""

import pytest
import torch

import mamba_hip

pytestmark = pytest.mark.gpu


def test_parameter_gradients_of_a_very_wide_row(dev):
    """2^27 + 40 columns: the sums of dw and db are over 2^28 + 80 columns, 16 a workgroup of
    256 threads, more threads than a grid of one workgroup each may have."""
    cols, mean, rstd = 2 ** 27 + 40, 0.25, 2.0
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    x, dy = (torch.randn(1, cols, generator=g, device=dev, dtype=torch.bfloat16) for _ in range(2))
    got = mamba_hip.layer_norm_bwd(dy, x, None, torch.full((1,), mean, device=dev), torch.full((1,), rstd, device=dev))
    assert torch.equal(got["dbias"], dy[0].float())  # one row: no sum
    assert torch.equal(got["dweight"], dy[0].float() * ((x[0].float() - mean) * rstd))
