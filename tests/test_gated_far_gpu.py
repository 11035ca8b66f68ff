"""Rows and states beyond 2^31 elements and 2^32 bytes: views of wide tensors give what their
copies give."""

import pytest
import torch

import mamba_hip

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_far_apart(dev, dtype):
    """The last rows lie past 2^32 bytes; the gradients too."""
    rows, d, st = 140, 70, (1 << 25) - 8
    if dtype == F32:
        rows = 100
    g = gen(1)
    cu = torch.tensor([0, 3, rows - 1], dtype=torch.int32, device=dev)
    wide = torch.empty(rows * st, dtype=dtype, device=dev).view(rows, st)  # 9.4 and 13.4 GB
    near = {k: torch.randn(rows, d, generator=g).to(dtype).to(dev) for k in "xrizw"}
    far = {}
    for k, (name, v) in enumerate(near.items()):
        far[name] = wide[:, st - 128 * (k + 1):][:, :d]
        far[name].copy_(v)
    A = (-0.2 * torch.rand(d, generator=g)).to(dev)
    carry, carry2 = torch.empty(-(-rows // 64), d, device=dev), torch.empty(-(-rows // 64), d, device=dev)
    want = mamba_hip.gated_scan_packed(near["x"], near["r"], near["i"], A, cu, near["z"], carry=carry)
    y = wide[:, :d]
    y.zero_()
    got = mamba_hip.gated_scan_packed(far["x"], far["r"], far["i"], A, cu, far["z"], carry=carry2, y=y)
    assert got is y and torch.equal(y, want) and torch.equal(carry[1:], carry2[1:])
    a = mamba_hip.gated_scan_packed_bwd(near["w"], near["x"], near["r"], near["i"], A, cu, carry, near["z"])
    b = mamba_hip.gated_scan_packed_bwd(far["w"], far["x"], far["r"], far["i"], A, cu, carry2, far["z"])
    assert all(torch.equal(a[k], b[k]) for k in ("dx", "dr", "di", "dz", "dA"))
    w = torch.rand(d, generator=g).to(dev)
    s = wide[:, 256:256 + d]
    for x, o in (((near["x"], near["r"]), None), ((far["x"], far["r"]), s)):
        out = mamba_hip.add_rms_norm(x[0], w, x[1], residual_out=o)
        want = out if o is None else want
    assert out[1] is s and torch.equal(out[0], want[0]) and torch.equal(s, want[1])


def test_far_slots(dev):
    """Slots past 2^31 elements of the cache."""
    d, n = 1 << 16, 33000  # 8.7 GB
    state = torch.empty(n, d, device=dev)
    g = gen(2)
    slots = torch.tensor([n - 1, 5, n - 2], dtype=torch.int32, device=dev)
    x, r, i = (torch.randn(3, d, generator=g).to(dev) for _ in range(3))
    A = (-0.2 * torch.rand(d, generator=g)).to(dev)
    start = torch.randn(3, d, generator=g).to(dev)
    state[slots.long()] = start
    want, small = None, start.clone()
    want = mamba_hip.gated_step_slots(x, r, i, A, small, None)
    assert torch.equal(mamba_hip.gated_step_slots(x, r, i, A, state, slots), want) and torch.equal(state[slots.long()], small)
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev)
    want = mamba_hip.gated_scan_packed(x, r, i, A, cu, state=small)
    assert torch.equal(mamba_hip.gated_scan_packed(x, r, i, A, cu, state=state, slots=slots), want) and torch.equal(state[slots.long()], small)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_products_of_rows_far_apart(dev, dtype):
    """Rows too far apart for one buffer's offsets are copied first; results lie as far apart."""
    rows, k, n, st = 130, 200, 90, 1 << 24
    g = gen(3)
    codes, scale = torch.randint(0, 16, (k, n), generator=g, dtype=torch.uint8).to(dev), torch.rand(-(-k // 64), n, generator=g).to(dev)
    w = mamba_hip.pack_linear_q4(codes, scale, None, 64)
    x = torch.randn(rows, k, generator=g).to(dtype).to(dev)
    wide = torch.empty(rows * st, dtype=dtype, device=dev).view(rows, st)  # 4.4 and 8.7 GB
    far, out = wide[:, st - k:], wide[:, 1:1 + n]
    far.copy_(x)
    assert torch.equal(mamba_hip.linear_q4(far, w, out=out), mamba_hip.linear_q4(x, w))
