"""Output gates of the type's lowest and highest values."""

import pytest
import torch

import gated_oracle as go
import mamba_hip
from packed_oracle import d as f64

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def cu(lens, dev):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_output_gates_of_the_lowest_value(dev, dtype):
    """silu of the type's lowest value is 0, whatever the state is; of its highest it is that value."""
    lens, d = [100, 40], 12
    n, g = sum(lens), gen(2)
    t = {k: torch.randn(n, d, generator=g).to(dtype).to(dev) for k in "xriz"}
    t["A"] = -0.1 * torch.rand(d, generator=g).to(dev)
    big = torch.finfo(dtype).max
    shut = torch.randint(0, 4, (n, d), generator=g) == 0
    t["z"][shut.to(dev)] = -big
    t["z"][5, 3], t["z"][6, 3] = -1e30, -1000.0
    shut[5, 3] = shut[6, 3] = True
    h0 = (8 * torch.randn(2, d, generator=g)).to(dev)  # states above 1: h z alone passes the range
    open_z = {**t, "z": torch.where(shut.to(dev), torch.zeros_like(t["z"]), t["z"])}
    c = cu(lens, dev)
    states = [h0.clone() for _ in range(2)]
    y = mamba_hip.gated_scan_packed(**t, cu_seqlens=c, state=states[0])
    want = mamba_hip.gated_scan_packed(**open_z, cu_seqlens=c, state=states[1])
    assert not y[shut.to(dev)].any() and torch.equal(y, want) and torch.equal(*states)
    # single tokens
    slots, cache = torch.arange(n, dtype=torch.int32, device=dev), [(8 * torch.randn(n, d, generator=gen(3))).to(dev) for _ in range(2)]
    y = mamba_hip.gated_step_slots(**t, state=cache[0], slots=slots)
    want = mamba_hip.gated_step_slots(**open_z, state=cache[1], slots=slots)
    assert not y[shut.to(dev)].any() and torch.equal(y, want) and torch.equal(*cache)
    # the gradients there are 0 but for what comes from later rows
    carry, dy = torch.empty(-(-n // 64), d, device=dev), torch.randn(n, d, generator=g).to(dtype).to(dev)
    mamba_hip.gated_scan_packed(**t, cu_seqlens=c, state=h0.clone(), carry=carry)
    got = mamba_hip.gated_scan_packed_bwd(dy, **t, cu_seqlens=c, carry=carry, initial_state=h0)
    for k, v in got.items():
        assert bool(torch.isfinite(v).all()), k
    assert not got["dz"][shut.to(dev)].any()
    # the highest: h z, within the range where |h| is at most one half
    t["z"][:] = big
    y = mamba_hip.gated_scan_packed(t["x"], t["r"], t["i"], torch.full_like(t["A"], -0.01), c, t["z"] * 0.5)
    plain = mamba_hip.gated_scan_packed(t["x"], t["r"], t["i"], torch.full_like(t["A"], -0.01), c)
    few = f64(plain).abs() < 0.5
    go.close(torch.where(few.to(dev), y, torch.zeros_like(y)), torch.where(few, f64(plain) * big / 2, torch.zeros_like(f64(plain))),
             f64(plain).abs() * big * (1 + 2.0 ** 14 * (dtype == BF16)), 4, "open")
