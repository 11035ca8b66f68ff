"""Decays so near to one that 1 - a^2 passes the smallest normal f32."""

import pytest
import torch

import gated_oracle as go
import mamba_hip

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def cu(lens, dev):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)


# (r, A); r is a bf16 too.  1 - a^2 = 2 |A| s(r) of the first is some 1e-36 and more, of the others below 2^-126 (and
# above 0 where the compiler keeps small numbers)
NORMAL = [(-80.0, -0.05), (-82.0, -0.05), (-80.0, -0.5), (-70.0, -1e-5), (-85.5, -6.0)]
BELOW = [(-85.5, -0.05), (-86.5, -0.05), (-87.0, -0.05), (-82.0, -0.001), (-84.0, -0.001), (-87.0, -0.001), (-87.0, -0.3), (-100.0, -0.05)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("z", [True, False])
@pytest.mark.parametrize("lens", [[70], [40, 1, 300, 0, 29]])
def test_weights_near_the_smallest_number(dev, dtype, z, lens):
    """Of states that are kept and take next to nothing in, all gradients are finite.  A weight below 2^-63 may
    be taken as 0 with what follows from it: that moves no output by more than rows x 2^-63 times its
    two other factors (x, dy, h and the gates' slopes stay below 2^6 each here)."""
    n, g = sum(lens), gen(1)
    pairs = NORMAL + BELOW
    A = torch.tensor([a for _, a in pairs] + [-1e-38, -4e-39]).to(dev)  # and tiny A with ordinary gates
    d = A.numel()
    t = {k: torch.randn(n, d, generator=g).to(dtype).to(dev) for k in "xri"}
    t["r"][:, :len(pairs)] = torch.tensor([r for r, _ in pairs], dtype=dtype, device=dev)
    if z:
        t["z"] = torch.randn(n, d, generator=g).to(dtype).to(dev)
    t["A"] = A
    h0, dhT = (torch.randn(len(lens), d, generator=g).to(dev) for _ in range(2))
    dy = torch.randn(n, d, generator=g).to(dtype).to(dev)
    carry, state = torch.empty(-(-n // 64), d, device=dev), h0.clone()
    c = cu(lens, dev)
    y = mamba_hip.gated_scan_packed(**t, cu_seqlens=c, state=state, carry=carry)
    got = mamba_hip.gated_scan_packed_bwd(dy, **t, cu_seqlens=c, carry=carry, initial_state=h0, d_final_state=dhT)
    for k, v in got.items():
        assert v is None or bool(torch.isfinite(v).all()), k
    ref = go.gated(lens, **t, h0=h0, dy=dy, dhT=dhT)
    k = go.gated_roundings(lens, t["r"], t["i"], t["A"], t.get("z"))
    few, least = len(NORMAL), n * 2.0 ** -63 * 2.0 ** 12 * 2.0 ** 23 / k  # go.close multiplies by k 2^-23
    for name, v in (("y", y), ("hT", state)):
        go.close(v, ref[name][0], ref[name][1] + least, k, name)
    for name in ("dx", "dr", "di") + (("dz",) if z else ()):
        go.close(got[name][:, :few], *(r[:, :few] for r in ref[name]), 2 * k, name)
        go.close(got[name][:, few:], ref[name][0][:, few:], ref[name][1][:, few:] + least, 2 * k, name)
    go.close(got["dA"][:few], *(r[:few] for r in ref["dA"]), 2 * k + n, "dA")
    go.close(got["d_initial_state"], ref["dh0"][0], ref["dh0"][1] + least, 2 * k, "dh0")
