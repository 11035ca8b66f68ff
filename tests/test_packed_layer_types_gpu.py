"""Types of the Mamba-1 layer's results, its own and under autocast."""

import pytest
import torch

import mamba_hip
import packed_oracle as po
from test_packed_layer_gpu import make, near, params, plain

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_token_keeps_its_type(dev, dtype):
    """Layer.step gives the type of its rows, with slots and without."""
    layer, x, _ = make(dev)
    ps, token = [po.d(t) for t in params(layer)], x[:3].to(dtype)
    want, _, _ = plain(layer, ps, po.d(token), [1] * 3)
    for slots in (None, torch.arange(3, dtype=torch.int32, device=dev)):
        y, _ = layer.step(token, layer.mixer.new_cache(3), slots)
        assert y.dtype == dtype
        # bf16 products and rows: some ten half steps of 2^-8 between x and y
        near(y, want, 1e-5 if dtype == F32 else 10 * 2.0 ** -8, str(slots))
