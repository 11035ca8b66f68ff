"""The gated recurrence's workspace is the caller's: one that is too small is refused before a
launch, and a call writes nothing behind the size that it asked for."""

import ctypes

import pytest
import torch

import mamba_hip
from mamba_hip import _lib
from mamba_hip.packed import _gated_args, _raw_stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,d", [(64, 5), (65, 300), (128, 5), (129, 300), (4500, 7)])
def test_workspace(dev, rows, d):
    g = torch.Generator().manual_seed(1)
    x, r, i = (torch.randn(rows, d, generator=g).to(dev) for _ in range(3))
    A, cu = -torch.rand(d, generator=g).to(dev), torch.tensor([0, rows], dtype=torch.int32, device=dev)
    want = mamba_hip.gated_scan_packed(x, r, i, A, cu)
    L, y = _lib.lib(), torch.empty_like(x)
    a = _gated_args(x, r, i, A, cu, None, None)
    a.y, a.y_st = y.data_ptr(), d
    need = L.mamba_gated_scan_workspace_size(ctypes.byref(a))
    assert (need == 0) == (rows <= 128)  # one tile of rows waits for none
    if need:
        assert L.mamba_gated_scan_fwd(ctypes.byref(a), None, 0, None) == 3
        ws = torch.full((need + 4096,), 77, dtype=torch.uint8, device=dev)
        assert L.mamba_gated_scan_fwd(ctypes.byref(a), ws.data_ptr(), need - 1, None) == 3
        assert L.mamba_gated_scan_fwd(ctypes.byref(a), ws.data_ptr() + 4, need, None) == 1
        for _ in range(2):  # what a call leaves there does not matter to the next
            assert L.mamba_gated_scan_fwd(ctypes.byref(a), ws.data_ptr(), need, _raw_stream(x)) == 0
            assert torch.equal(y, want) and bool((ws[need:] == 77).all())
