"""Values that are not finite in the packed scan and the slot steps: they reach what the
formulas say, and nothing else."""

import pytest
import torch

import mamba_hip
import packed_oracle as po
from test_packed_gpu import cu, gen, oracle_args, scan_inputs

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("name", ["delta", "delta_bias"])
def test_nan_step_is_not_a_number(dev, name, dtype):
    """A NaN in delta reaches its channel from its row on, one in delta_bias its whole
    channel, and nothing else: in chunks, in whole sequences, and in the gradients."""
    lens, d, n = [90, 40, 200], 20, 16
    t = scan_inputs(lens, d, n, dtype, dev, seed=40)
    c, dy = cu(lens, dev), torch.ones(sum(lens), d, dtype=dtype, device=dev)
    hit = torch.zeros(sum(lens), d, dtype=torch.bool, device=dev)  # rows and channels that are no number in y
    ends = torch.zeros(3, d, dtype=torch.bool, device=dev)
    bad = {k: v.clone() for k, v in t.items()}
    if name == "delta":
        bad["delta"][100, 3] = NAN
        hit[100:130, 3] = ends[1, 3] = True
        back = torch.zeros_like(hit)
        back[90:130, 3] = True  # ddelta: the state after the row, the gradient before it
    else:
        bad["delta_bias"][3] = NAN
        hit[:, 3] = ends[:, 3] = True
        back = hit
    for most in (0, 96):
        state, want = torch.zeros(3, d, n, device=dev), torch.zeros(3, d, n, device=dev)
        clean = mamba_hip.mamba1_scan_packed(**t, cu_seqlens=c, delta_softplus=True, state=want, max_seqlen=most)
        y = mamba_hip.mamba1_scan_packed(**bad, cu_seqlens=c, delta_softplus=True, state=state, max_seqlen=most)
        assert torch.equal(y.isnan(), hit) and torch.equal(y[~hit], clean[~hit]), most
        assert torch.equal(state.isnan(), ends[..., None].expand_as(state)) and torch.equal(state[~ends], want[~ends]), most
    want = mamba_hip.mamba1_scan_packed_bwd(dy, **t, cu_seqlens=c, delta_softplus=True)
    g = mamba_hip.mamba1_scan_packed_bwd(dy, **bad, cu_seqlens=c, delta_softplus=True)
    assert torch.equal(g["ddelta"].isnan(), back) and torch.equal(g["ddelta"][~back], want["ddelta"][~back])
    assert torch.equal(g["dz"].isnan(), hit) and torch.equal(g["dz"][~hit], want["dz"][~hit])
    rest = torch.arange(d, device=dev) != 3
    for k in ("dA", "dD", "d_delta_bias"):
        assert torch.equal(g[k][rest], want[k][rest]), k
    assert g["dA"][3].isnan().all() and g["d_delta_bias"][3].isnan()


@pytest.mark.parametrize("n", [16, 12])
@pytest.mark.parametrize("name", ["delta", "delta_bias"])
def test_nan_step_of_a_token(dev, name, n):
    b, d = 5, 70
    t = scan_inputs([1] * b, d, n, F32, dev, seed=41)
    bad = {k: v.clone() for k, v in t.items()}
    hit = torch.zeros(b, d, dtype=torch.bool, device=dev)
    if name == "delta":
        bad["delta"][2, 7] = NAN
        hit[2, 7] = True
    else:
        bad["delta_bias"][7] = NAN
        hit[:, 7] = True
    slots = torch.randperm(b, generator=gen(42)).to(device=dev, dtype=torch.int32)
    state = torch.randn(b, d, n, generator=gen(43)).to(dev)
    want = state.clone()
    clean = mamba_hip.scan_step_slots(**t, state=want, slots=slots, delta_softplus=True)
    y = mamba_hip.scan_step_slots(**bad, state=state, slots=slots, delta_softplus=True)
    assert torch.equal(y.isnan(), hit) and torch.equal(y[~hit], clean[~hit])
    got, want = state[slots.long()], want[slots.long()]
    assert torch.equal(got.isnan(), hit[..., None].expand_as(got)) and torch.equal(got[~hit], want[~hit])

def like(got, ref, what):
    """The same infinities, the same places that are no number, finite elsewhere."""
    g = po.d(got)
    assert torch.equal(g.isnan(), ref.isnan()), (what, "nan", int(g.isnan().sum()), int(ref.isnan().sum()))
    assert torch.equal(g == INF, ref == INF) and torch.equal(g == -INF, ref == -INF), what


def positive(lens, d, n, dev, seed):
    """Every input that multiplies is positive, so that infinities have one sign, and the
    decay of a sequence stays far from 0, so that an infinite state stays one."""
    t = scan_inputs(lens, d, n, F32, dev, seed=seed)
    for k in ("u", "B", "C", "D", "z"):
        t[k] = t[k].abs() + 0.1
    t["delta"] = t["delta"].clamp(-1, 1)
    t["delta_bias"] = t["delta_bias"].clamp(-6, -4)
    return t


@pytest.mark.parametrize("n", [16, 1, 5, 12, 20, 33])
def test_infinite_input(dev, n):
    """An infinite u makes its channel infinite from its row on, whatever the states are padded to."""
    lens, d = [20, 60, 9], 3
    t = positive(lens, d, n, dev, 44)
    t["u"][30, 1] = INF
    dy, c = torch.ones(sum(lens), d, device=dev), cu(lens, dev)
    ref = po.scan(lens, dy=dy, **oracle_args(t, True))
    assert ref["y"][0].isinf().sum() == 50 and not ref["y"][0].isnan().any()
    for most in (0, 60):
        state = torch.zeros(3, d, n, device=dev)
        like(mamba_hip.mamba1_scan_packed(**t, cu_seqlens=c, delta_softplus=True, state=state, max_seqlen=most), ref["y"][0], "y")
        like(state, ref["hT"][0], "state")
    g = mamba_hip.mamba1_scan_packed_bwd(dy, **t, cu_seqlens=c, delta_softplus=True)
    for k in ("du", "ddelta", "dz", "dB", "dC", "dA", "dD"):
        like(g[k], ref[k][0], k)

@pytest.mark.parametrize("name,n", [("B", 16), ("C", 16), ("B", 12), ("C", 64), ("C", 5)])
def test_infinite_projection(dev, name, n):
    """An infinite B or C: the channels that the last workgroup is padded with add nothing to
    dB and dC."""
    lens, d = [20, 60, 9], 3
    t = positive(lens, d, n, dev, 45)
    t[name][30, n - 1] = INF
    dy, c = torch.ones(sum(lens), d, device=dev), cu(lens, dev)
    ref = po.scan(lens, dy=dy, **oracle_args(t, True))
    assert ref["dC" if name == "B" else "dB"][0].isinf().any()
    like(mamba_hip.mamba1_scan_packed(**t, cu_seqlens=c, delta_softplus=True), ref["y"][0], "y")
    g = mamba_hip.mamba1_scan_packed_bwd(dy, **t, cu_seqlens=c, delta_softplus=True)
    for k in ("du", "ddelta", "dz", "dB", "dC", "dA", "dD"):
        like(g[k], ref[k][0], k)
