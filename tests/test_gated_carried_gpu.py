"""States carried over groups of tiles, between sequences of a cache: each channel has a bound of its own, so that
an error of a slow channel is not hidden by what a steep one may be off by.

A row multiplies what it takes over by its decay and adds its term: 4 + |w| (6 + 2 |r|) roundings of
2^-23 (w = A s(r): the decay's own).  The error obeys the recurrence itself, e_t = a_t e_{t-1} + that many
roundings of the sum of the absolute values m_t; what is around it (weights, gates, their slopes) has at
most 40 + 4 (|r| + |i| + |z|) roundings."""

import pytest
import torch

import mamba_hip
from packed_oracle import F64, half_step
from packed_oracle import d as f64

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def within(got, ref, err, what):
    tol = half_step(got.dtype) * ref.abs() * (1 + 2 ** -8) + err + 1e-37
    off = (f64(got) - ref).abs()
    assert bool((off <= tol).all()), (what, float((off / tol).max()))


def walk(lens, a, add, start, back=False):
    """v_t = a_t v_{t-1} + add_t from start [s, d] (back: v_t = add_t + a_{t+1} v_{t+1} from start at
    the end, as it stands there): (v, what each row takes over, what is left behind the last one)."""
    v, before, left, n = torch.zeros_like(add), torch.zeros_like(add), start.clone(), 0
    for s, length in enumerate(lens):
        for t in (reversed(range(n, n + length)) if back else range(n, n + length)):
            before[t] = left[s]
            if back:
                v[t] = add[t] + left[s]
                left[s] = a[t] * v[t]
            else:
                left[s] = v[t] = a[t] * left[s] + add[t]
        n += length
    return v, before, left


LENS = {"groups": [2500, 1, 0, 3900, 200], "far": [9000], "short": [130, 1, 64, 63]}


@pytest.mark.parametrize("name", LENS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("z", [True, False])
def test_carried(dev, name, dtype, z):
    lens, g = LENS[name], gen(1)
    n = sum(lens)
    # states that last thousands of rows beside states that last one
    A = -torch.tensor([1e-5, 2e-4, 0.002, 0.02, 0.1, 0.13, 0.5, 3.0, 6.0])
    d, s = A.numel(), len(lens)
    t = {k: torch.randn(n, d, generator=g).to(dtype) for k in ("x", "r", "i", "z", "dy")}
    if not z:
        t["z"] = None
    h0, dhT = (torch.randn(s, d, generator=g) for _ in range(2))
    slots = torch.randperm(s + 2, generator=g)[:s].to(torch.int32)
    cache = torch.randn(s + 2, d, generator=g)
    cache[slots.long()] = h0
    c = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    on = {k: None if v is None else v.to(dev) for k, v in t.items()}
    state, carry, Ad = cache.to(dev), torch.empty(-(-n // 64), d, device=dev), A.to(dev)
    y = mamba_hip.gated_scan_packed(on["x"], on["r"], on["i"], Ad, c, on["z"], state=state, slots=slots.to(dev))
    first = h0.to(dev)
    mamba_hip.gated_scan_packed(on["x"], on["r"], on["i"], Ad, c, on["z"], state=first.clone(), carry=carry)
    got = mamba_hip.gated_scan_packed_bwd(on["dy"], on["x"], on["r"], on["i"], Ad, c, carry, on["z"], first, dhT.to(dev))

    X, R, I, Z, G, A = f64(t["x"]), f64(t["r"]), f64(t["i"]), f64(t["z"]), f64(t["dy"]), f64(A)
    step = 2.0 ** -23
    sr, si = torch.sigmoid(R), torch.sigmoid(I)
    w = A * sr
    a, m, u = torch.exp(w), torch.sqrt(-torch.expm1(2 * w)), si * X
    sz = None if Z is None else torch.sigmoid(Z)
    gate = torch.ones_like(u) if Z is None else Z * sz
    own = (4 + w.abs() * (6 + 2 * R.abs())) * step
    base = (40 + 4 * (R.abs() + I.abs() + (0 if Z is None else Z.abs()))) * step
    none = torch.zeros(s, d, dtype=F64)
    h, hb, hT = walk(lens, a, m * u, f64(h0))
    mag, magb, _ = walk(lens, a, m * u.abs(), f64(h0).abs())
    eh, ehb, ehT = walk(lens, a, (own + base) * mag, none)
    within(y, h * gate, (eh + base * mag) * gate.abs(), "y")
    live = [k for k, v in enumerate(lens) if v]
    within(state[slots[live].long().to(dev)], hT[live], ehT[live], "state")
    others = [k for k in range(s + 2) if k not in slots[live].tolist()]
    assert torch.equal(state.cpu()[others], cache[others])
    dh, _, dh0 = walk(lens, a, G * gate, f64(dhT), True)
    dmag, _, dmag0 = walk(lens, a, (G * gate).abs(), f64(dhT).abs(), True)
    ed, _, ed0 = walk(lens, a, (own + base) * dmag, none, True)
    within(got["d_initial_state"], dh0, ed0 + (own.amax(0) + base.amax(0)) * dmag0, "d_initial_state")
    within(got["dx"], dh * m * si, (ed + base * dmag) * m * si, "dx")
    k = m * u * torch.sigmoid(-I)
    within(got["di"], dh * k, (ed + base * dmag) * k.abs(), "di")
    pull = u * a * a / m
    e, ah = dh * (a * hb - pull), a * magb + pull.abs()
    ee = ed * ah + dmag * (a * ehb + (base + own) * ah)
    kr = w.abs() * torch.sigmoid(-R)
    within(got["dr"], e * w * torch.sigmoid(-R), (ee + base * dmag * ah) * kr, "dr")
    if z:
        slope = sz * (1 + Z * torch.sigmoid(-Z))
        within(got["dz"], G * h * slope, (eh + base * mag) * (G * slope).abs() + base * mag * G.abs() * sz * (1 + Z.abs()), "dz")
    # a sum over the rows: of 8 in turn in a lane, over the waves, the tiles in 16 runs of 4
    within(got["dA"], (e * sr).sum(0), ((ee + base * dmag * ah) * sr).sum(0) + (24 + n / 64 / 64) * step * (dmag * ah * sr).sum(0), "dA")
