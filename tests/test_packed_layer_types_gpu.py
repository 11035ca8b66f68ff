"""Types of the Mamba-1 layer's results, its own and under autocast."""

import pytest
import torch

import mamba_hip
import packed_oracle as po
from test_packed_layer_gpu import LENS, NAMES, make, near, params, plain

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


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

def test_dropout_under_autocast(dev):
    """f32 rows whose products autocast makes bf16: the result is f32 with an rng as it is
    without one, and everything gets its gradient."""
    layer, x, cu = make(dev, p=0.3)
    leaves = [t.requires_grad_() for t in params(layer)] + [x.requires_grad_()]
    rng = torch.tensor([5, 9], device=dev)
    with torch.autocast("cuda", BF16):
        assert layer.forward_packed(x, cu).dtype == F32
        y = layer.forward_packed(x, cu, rng=rng, offset=2)
    assert y.dtype == F32
    keep = po.philox_kept(x.numel(), 0.3, 5, 11).reshape(x.shape).to(F64)
    # bf16 products and rows: some ten half steps of 2^-8 between x and y
    near(y, plain(layer, [po.d(t) for t in leaves[:-1]], po.d(x), LENS, keep)[0], 10 * 2.0 ** -8, "y")
    for name, g, t in zip(NAMES + ("norm_w", "norm_b", "x"), torch.autograd.grad(y.sum(), leaves), leaves):
        assert g.dtype == t.dtype and torch.isfinite(g).all() and g.any(), name
