"""What lies behind a packed 4-bit weight is no part of a product: with bytes of all ones there (NaN as
a scale, and as a code of rows that are not there) the results keep their bits."""

import pytest
import torch

import mamba_hip

pytestmark = pytest.mark.gpu
BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


# fewer blocks of k than a workgroup's waves and their turns take, and k that is walked
@pytest.mark.parametrize("k", [1, 32, 128, 130, 520, 1100, 3200, 5200, 8000])
@pytest.mark.parametrize("group,zero,sdtype", [(32, True, F32), (64, False, BF16), (128, True, BF16), (64, False, F32)])
@pytest.mark.parametrize("dtype", [F32, BF16, I8])
def test_behind_the_weight(dev, k, group, zero, sdtype, dtype):
    g, n = gen(k), 37
    groups = -(-k // group)
    codes = torch.randint(0, 16, (k, n), generator=g, dtype=torch.uint8).to(dev)
    scale = ((0.5 + torch.rand(groups, n, generator=g)) * 0.02).to(sdtype).to(dev)
    z = torch.randint(0, 16, (groups, n), generator=g, dtype=torch.uint8).to(dev) if zero else None
    w = mamba_hip.pack_linear_q4(codes, scale, z, group)
    size = w.data.numel()
    wide = torch.full((size + (1 << 20),), 0xff, dtype=torch.uint8, device=dev)
    wide[:size] = w.data
    front = mamba_hip.PackedQ4(w.d_in, w.d_out, w.group, w.scale_dtype, w.has_zero, wide[:size])
    for rows in (1, 19, 70):
        if dtype == I8:
            x, xs = torch.randint(-127, 128, (rows, k), generator=g, dtype=I8).to(dev), torch.rand(rows, generator=g).to(dev)
        else:
            x, xs = torch.randn(rows, k, generator=g).to(dtype).to(dev), None
        y = mamba_hip.linear_q4(x, front, x_scale=xs, dtype=F32)
        dense = (codes.cpu().double() - (8 if z is None else z.cpu().double().repeat_interleave(group, 0)[:k])) * scale.cpu().double().repeat_interleave(group, 0)[:k]
        want = x.cpu().double() @ dense
        if xs is not None:
            want *= xs.cpu().double()[:, None]
        assert bool(torch.isfinite(y).all()), rows
        assert float((y.cpu().double() - want).norm()) <= 1e-5 * float(want.norm()), rows  # no other block's values
        assert torch.equal(y, mamba_hip.linear_q4(x, w, x_scale=xs, dtype=F32)), rows


def test_the_last_scales_may_be_infinite(dev):
    """A column's last group with an infinite scale gives what that is times the group's sum, and a NaN
    nowhere: no block behind the last takes its values."""
    k, n = 130, 20
    g = gen(3)
    codes = torch.randint(9, 16, (k, n), generator=g, dtype=torch.uint8).to(dev)
    scale = torch.rand(3, n, generator=g).to(dev)
    scale[2, 4] = float("inf")
    w = mamba_hip.pack_linear_q4(codes, scale, None, 64)
    for dtype in (F32, BF16):
        y = mamba_hip.linear_q4(torch.ones(3, k, dtype=dtype, device=dev), w, dtype=F32)
        assert bool((y[:, 4] == float("inf")).all()) and bool(torch.isfinite(y[:, [c for c in range(n) if c != 4]]).all())
