"""The packed scan over more chunks than walk by themselves (128): the carries of a kernel
of their own, forward and backward, for every number of padded states.  The sequences
are of chunk-like lengths, so that most cross a border and the bound on roundings (which
grows with the longest) stays small."""

import ctypes

import pytest
import torch

import mamba_hip
import packed_oracle as po
from mamba_hip import packed
from test_packed_gpu import cu, gen, oracle_args, roundings, scan_inputs, strided

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
LENS = torch.randint(20, 150, (90,), generator=gen(50)).tolist() + [0, 1, 220, 64, 128] + [100] * 6


@pytest.mark.parametrize("n,dtype", [(16, F32), (16, BF16), (32, F32), (64, BF16), (6, BF16), (40, F32)])
def test_many_chunks(dev, n, dtype):
    lens, d, pad = LENS, 7, 5
    t = scan_inputs(lens, d, n, dtype, dev, seed=51, pad=pad)
    c, count = cu(lens, dev), len(lens)
    args = packed._scan_args(t["u"], t["delta"], t["A"], t["B"], t["C"], c, t["D"], t["z"], t["delta_bias"], True, 0)
    padded = 8 if n <= 8 else 16 if n <= 16 else 32 if n <= 32 else 64
    # the workspace holds two states of every chunk
    assert mamba_hip.lib().mamba1_scan_packed_workspace_size(ctypes.byref(args)) > 129 * 2 * 4 * d * padded
    g = gen(52)
    h0, dhT = (torch.randn(count, d, n, generator=g).to(dev) for _ in range(2))
    dy = strided(g, sum(lens) + pad, d, dtype, dev)
    ref, k = po.scan(lens, h0=h0, dy=dy, dhT=dhT, **oracle_args(t, True)), roundings(lens)
    slots = torch.randperm(count, generator=g).to(dev)
    state = torch.empty_like(h0)
    state[slots] = h0
    y = mamba_hip.mamba1_scan_packed(**t, cu_seqlens=c, delta_softplus=True, state=state, slots=slots.to(torch.int32))
    po.close(y, *ref["y"], k, "y")
    po.close(state[slots], *ref["hT"], k, "state")
    got = mamba_hip.mamba1_scan_packed_bwd(dy, **t, cu_seqlens=c, delta_softplus=True, initial_state=h0, d_final_state=dhT)
    for name in ("du", "ddelta", "dz", "dB", "dC"):
        po.close(got[name], *ref[name], 2 * k, name)
    po.close(got["d_initial_state"], *ref["dh0"], 2 * k, "d_initial_state")
    for name, of in (("dA", "dA"), ("dD", "dD"), ("d_delta_bias", "dbias")):  # sums over the rows besides
        po.close(got[name], *ref[of], 2 * k + sum(lens), name)
