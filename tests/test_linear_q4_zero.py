"""Zero points of 4-bit weights: 0 to 16 are held (formats that keep them less one give 1 to 16), larger
ones are refused, and give a NaN where only the C entry sees them."""

import ctypes

import pytest
import torch

import mamba_hip
from mamba_hip import _lib
from mamba_hip.packed import _raw_stream

BF16, F32, I8, U8 = torch.bfloat16, torch.float32, torch.int8, torch.uint8


@pytest.mark.parametrize("value", [17, 31, 32, 255])
def test_larger_ones_are_refused(value):
    zero = torch.full((2, 10), 8, dtype=U8)
    zero[1, 7] = value
    with pytest.raises(mamba_hip.MambaHipError, match="zero points"):
        mamba_hip.pack_linear_q4(torch.zeros(64, 10, dtype=U8), torch.ones(2, 10), zero)


@pytest.mark.gpu
@pytest.mark.parametrize("sdtype", [F32, BF16])
@pytest.mark.parametrize("k", [128, 8192])  # rows held and k walked
def test_each_zero_point(dev, k, sdtype):
    """A column for each, every code in it: whole numbers, exact in every type."""
    n = 17
    codes = (torch.arange(k)[:, None] + 3 * torch.arange(n)[None]).remainder(16).to(U8).to(dev)
    zero = (torch.arange(n)[None] + 5 * torch.arange(k // 64)[:, None]).remainder(17).to(U8).to(dev)
    w = mamba_hip.pack_linear_q4(codes, torch.ones(k // 64, n, dtype=sdtype, device=dev), zero)
    want = codes.float() - zero.float().repeat_interleave(64, 0)
    at = torch.arange(0, k, k // 128)
    x = torch.zeros(128, k)
    x[torch.arange(128), at] = 1
    for dtype in (BF16, F32):
        assert torch.equal(mamba_hip.linear_q4(x.to(dtype).to(dev), w, dtype=F32), want[at.to(dev)])
    one = torch.ones(128, device=dev)
    assert torch.equal(mamba_hip.linear_q4(x.to(I8).to(dev), w, x_scale=one, dtype=F32), want[at.to(dev)])


@pytest.mark.gpu
@pytest.mark.parametrize("sdtype", [F32, BF16])
def test_larger_ones_through_the_c_entry(dev, sdtype):
    k, n = 128, 40
    codes = torch.full((k, n), 9, dtype=U8, device=dev)
    scale = torch.ones(2, n, dtype=sdtype, device=dev)
    zero = torch.full((2, n), 8, dtype=U8, device=dev)
    w = mamba_hip.pack_linear_q4(codes, scale, zero)
    zero[1, 5], zero[0, 39] = 17, 255
    c = _lib.Q4Weight()
    w._fill(c)
    assert _lib.lib().mamba_linear_q4_pack(ctypes.byref(c), codes.data_ptr(), scale.data_ptr(), zero.data_ptr(), w.data.data_ptr(), _raw_stream(codes)) == 0
    bad = [i in (5, 39) for i in range(n)]
    for x, xs in ((torch.ones(3, k, device=dev), None), (torch.ones(3, k, dtype=I8, device=dev), torch.ones(3, device=dev))):
        y = mamba_hip.linear_q4(x, w, x_scale=xs, dtype=F32)
        assert y.isnan().all(0).tolist() == bad and bool((y[:, ~torch.tensor(bad)] == k).all())


@pytest.mark.gpu
def test_captured(dev):
    """Laid out in a graph, again from codes and zero points that have changed."""
    k, n = 128, 40
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 16, (k, n), generator=g, dtype=U8).to(dev)
    zero, scale = torch.randint(0, 17, (2, n), generator=g, dtype=U8).to(dev), torch.rand(2, n, generator=g).to(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w = mamba_hip.pack_linear_q4(codes, scale, zero)
    for turn in range(3):
        codes.copy_((codes + turn).remainder(16))
        zero.copy_((zero + turn).remainder(17))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w.data, mamba_hip.pack_linear_q4(codes, scale, zero).data)
