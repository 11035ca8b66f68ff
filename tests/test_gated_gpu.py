"""The gated linear recurrence over packed sequences, its gradients and its slot step against
plain 64-bit forms (gated_oracle), where they can go wrong: empty and one-row sequences,
sequences that cross tiles and groups of tiles, odd widths, strided rows, padding rows
that hold NaN, slots out of range, decays of exactly one, captured and concurrent calls."""

import pytest
import torch

import gated_oracle as go
import mamba_hip
from packed_oracle import d as f64

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

LENS = {
    "none": [],
    "empties": [0, 0, 0],
    "one": [1],
    "short": [7],
    "mixed": [0, 1, 130, 0, 63, 200, 5, 0],
    "borders": [64, 64, 128, 1, 127, 256],
    "long": [700],
    "tokens": [1] * 70,
    "groups": [2500, 1, 0, 3900, 200],  # tiles' groups crossed within a sequence, several times
    "far": [9000],
    "crowd": [3] * 20 + [0] * 500 + [1, 0] * 100 + [40] + [0] * 1000 + [2, 90],  # many in a tile, and long runs of empty ones
}


def cu(lens, dev):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist() if lens else [0], dtype=torch.int32, device=dev)


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def strided(g, rows, cols, dtype, dev, left=3, right=2):
    """[rows, cols] in the middle of wider rows."""
    return torch.randn(rows, left + cols + right, generator=g).to(dtype).to(dev)[:, left:left + cols]


def inputs(lens, d, dtype, dev, seed=0, pad=0, z=True, steep=False):
    g, rows = gen(seed), sum(lens) + pad
    t = dict(x=strided(g, rows, d, dtype, dev), r=strided(g, rows, d, dtype, dev, 1, 0), i=strided(g, rows, d, dtype, dev, 0, 4))
    if z:
        t["z"] = strided(g, rows, d, dtype, dev)
    # one in four channels keeps little of its state a row, so that the exponential's far side is used too
    a = torch.rand(d, generator=g)
    t["A"] = -torch.where(torch.arange(d) % 4 == 1, 6 * a, 0.001 + (0.5 if steep else 0.05) * a).to(dev)
    if pad:
        for k in ("x", "r", "i", "z"):
            if k in t:
                t[k][-pad:] = float("nan")
    return t


def roundings(lens, t):
    return go.gated_roundings(lens, t["r"], t["i"], t["A"], t.get("z"))


CASES = [("one", 1, F32, 0, True), ("short", 5, BF16, 2, False), ("mixed", 70, F32, 3, True), ("mixed", 64, BF16, 0, True),
         ("borders", 37, F32, 0, True), ("borders", 129, BF16, 70, False), ("long", 65, BF16, 1, False), ("tokens", 40, F32, 0, True),
         ("mixed", 130, BF16, 3, True), ("mixed", 257, F32, 0, False), ("groups", 6, F32, 5, True), ("groups", 9, BF16, 0, False),
         ("far", 3, BF16, 0, True), ("none", 4, F32, 3, True), ("empties", 4, BF16, 3, True), ("crowd", 65, F32, 2, True),
         ("crowd", 9, BF16, 0, False)]


@pytest.mark.parametrize("name,d,dtype,pad,z", CASES)
def test_forward(dev, name, d, dtype, pad, z):
    lens = LENS[name]
    t = inputs(lens, d, dtype, dev, pad=pad, z=z)
    k = roundings(lens, t)
    slots = torch.randperm(len(lens) + 3, generator=gen(1))[:len(lens)].to(torch.int32)
    state = torch.randn(len(lens) + 3, d, generator=gen(2)).to(dev)
    ref = go.gated(lens, **t, h0=state.cpu()[slots.long()])
    before = state.clone()
    y = mamba_hip.gated_scan_packed(**t, cu_seqlens=cu(lens, dev), state=state, slots=slots.to(dev))
    go.close(y, *ref["y"], k, "y")
    go.close(state[slots.long()], *ref["hT"], k, "state")
    others = [i for i in range(len(lens) + 3) if i not in slots.tolist()]
    assert torch.equal(state[others], before[others])
    again = before.clone()
    assert torch.equal(y, mamba_hip.gated_scan_packed(**t, cu_seqlens=cu(lens, dev), state=again, slots=slots.to(dev)))
    assert torch.equal(again, state)
    # without a state: from zero, nothing kept
    ref = go.gated(lens, **t)
    go.close(mamba_hip.gated_scan_packed(**t, cu_seqlens=cu(lens, dev)), *ref["y"], k, "y from zero")


@pytest.mark.parametrize("name,d,dtype,pad,z", CASES)
def test_backward(dev, name, d, dtype, pad, z):
    lens = LENS[name]
    t = inputs(lens, d, dtype, dev, seed=3, pad=pad, z=z)
    g = gen(4)
    h0, dhT = (torch.randn(len(lens), d, generator=g).to(dev) for _ in range(2))
    dy = strided(g, sum(lens) + pad, d, dtype, dev)
    if pad:
        dy[-pad:] = float("nan")
    k = 2 * roundings(lens, t)
    for start in (None, h0):
        back = None if start is None else dhT
        carry = torch.full((-(-t["x"].shape[0] // 64), d), float("nan"), device=dev)
        mamba_hip.gated_scan_packed(**t, cu_seqlens=cu(lens, dev), state=None if start is None else start.clone(), carry=carry)
        ref = go.gated(lens, **t, h0=start, dy=dy, dhT=back)
        call = lambda: mamba_hip.gated_scan_packed_bwd(dy, **t, cu_seqlens=cu(lens, dev), carry=carry, initial_state=start, d_final_state=back)  # noqa: E731, B023
        got = call()
        for key in ("dx", "dr", "di") + (("dz",) if z else ()):
            go.close(got[key], *ref[key], k, key)
        go.close(got["dA"], *ref["dA"], k + sum(lens), "dA")  # a sum over the rows besides
        assert z or got["dz"] is None
        if start is None:
            assert got["d_initial_state"] is None
        else:
            go.close(got["d_initial_state"], *ref["dh0"], k, "d_initial_state")
        again = call()
        for key, v in got.items():
            assert v is None or torch.equal(v, again[key]), key


def test_gradient_by_differences(dev):
    """The gradient along a direction against the difference quotient of the 64-bit form."""
    lens = [3, 70, 0, 20]
    t = inputs(lens, 6, F32, dev, seed=5, steep=True)
    dy = torch.randn(sum(lens), 6, generator=gen(6)).to(dev)
    carry = torch.empty(2, 6, device=dev)
    mamba_hip.gated_scan_packed(**t, cu_seqlens=cu(lens, dev), carry=carry)
    got = mamba_hip.gated_scan_packed_bwd(dy, **t, cu_seqlens=cu(lens, dev), carry=carry)
    for k, gk in dict(x="dx", r="dr", i="di", A="dA", z="dz").items():
        v = torch.randn(t[k].shape, generator=gen(7), dtype=torch.float64)
        if k == "A":
            v = v * f64(t["A"]).abs()  # a step that keeps A below 0, and the quotient's error small beside it
        step = 1e-5

        def objective(sign):
            moved = {key: f64(x) for key, x in t.items()}
            moved[k] = moved[k] + sign * step * v
            return float((go.gated(lens, **moved)["y"][0] * f64(dy)).sum())

        quotient = (objective(1) - objective(-1)) / (2 * step)
        along = float((f64(got[gk]) * v).sum())
        # the quotient is off by step^2 of third derivatives, the gradient by f32 roundings
        assert abs(along - quotient) <= 1e-4 * (abs(quotient) + float((f64(got[gk]).abs() * v.abs()).sum())), (k, along, quotient)


@pytest.mark.parametrize("name,dtype", [("mixed", F32), ("groups", BF16)])
def test_autograd(dev, name, dtype):
    lens, d = LENS[name], 24
    t = inputs(lens, d, dtype, dev, seed=8)
    h0 = torch.randn(len(lens), d, generator=gen(9)).to(dev)
    leaves = {k: v.detach().clone().requires_grad_() for k, v in t.items()}
    h0_ = h0.clone().requires_grad_()
    y, hT = mamba_hip.gated_scan_packed_autograd(**leaves, cu_seqlens=cu(lens, dev), initial_state=h0_)
    dy, dhT = torch.randn(y.shape, generator=gen(10)).to(dtype).to(dev), torch.randn(hT.shape, generator=gen(11)).to(dev)
    grads = torch.autograd.grad((y, hT), [*leaves.values(), h0_], (dy, dhT))
    ref = go.gated(lens, **t, h0=h0, dy=dy, dhT=dhT)
    k = 2 * roundings(lens, t)
    go.close(y, *ref["y"], k, "y")
    go.close(hT, *ref["hT"], k, "hT")
    for key, got in zip([*leaves, "h0"], grads):
        go.close(got, *ref["d" + key], k + (sum(lens) if key == "A" else 0), key)
    # one output alone, an expanded gradient
    y, hT = mamba_hip.gated_scan_packed_autograd(**leaves, cu_seqlens=cu(lens, dev))
    one = torch.autograd.grad(y.sum(), leaves["x"])[0]
    ref = go.gated(lens, **t, dy=torch.ones_like(dy))
    go.close(one, *ref["dx"], k, "dx of a sum")
    y, hT = mamba_hip.gated_scan_packed_autograd(**leaves, cu_seqlens=cu(lens, dev))
    one = torch.autograd.grad(hT, leaves["i"], dhT)[0]
    ref = go.gated(lens, **t, dy=torch.zeros_like(dy), dhT=dhT)
    go.close(one, *ref["di"], k, "di of the states")


def test_open_and_shut_gates(dev):
    """A decay of exactly one (A = 0, or a gate shut so far that A s(r) is 0) keeps the state
    and takes nothing in; gradients stay finite there.  A decay of nothing takes all in."""
    lens, d = [70], 8
    t = inputs(lens, d, F32, dev, seed=12)
    t["A"][0] = 0.0
    t["r"][:, 1] = -200.0
    t["A"][2], t["r"][:, 2] = -1e5, 4.0  # exp underflows
    t["i"][:, 3], t["i"][:, 4] = 200.0, -200.0
    h0 = torch.randn(1, d, generator=gen(13)).to(dev)
    carry, state = torch.empty(2, d, device=dev), h0.clone()
    t["z"] = None
    y = mamba_hip.gated_scan_packed(**t, cu_seqlens=cu(lens, dev), state=state, carry=carry)
    assert torch.equal(y[:, 0], h0[0, 0].expand(70)) and torch.equal(y[:, 1], h0[0, 1].expand(70))
    go.close(y[:, 2], f64(t["i"][:, 2]).sigmoid() * f64(t["x"][:, 2]), (f64(t["i"][:, 2]).sigmoid() * f64(t["x"][:, 2])).abs(), 20, "taken in")
    dy = torch.randn(70, d, generator=gen(14)).to(dev)
    got = mamba_hip.gated_scan_packed_bwd(dy, **t, cu_seqlens=cu(lens, dev), carry=carry, initial_state=h0)
    for key in ("dx", "dr", "di", "dA", "d_initial_state"):
        assert bool(torch.isfinite(got[key]).all()), key
    assert not got["dx"][:, :2].any() and not got["dr"][:, :2].any() and not got["di"][:, :2].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_nonfinite_values_stay_in_their_sequence_and_channel(dev, dtype):
    """A NaN or an infinity in one sequence's row reaches its own channel's later rows and
    gradients, and no other sequence's, though tiles hold rows of several."""
    lens, d = [100, 300, 90, 2200, 40], 10
    t = inputs(lens, d, dtype, dev, seed=15)
    clean = {k: v.clone() for k, v in t.items()}
    starts = [0, 100, 400, 490, 2690]
    t["x"][150, 2] = float("nan")
    t["x"][500, 3] = float("inf")
    t["r"][2700, 4] = float("nan")
    t["r"][120, 5] = float("nan")
    if dtype == F32:  # a NaN of all ones, as uninitialised memory holds
        t["r"].view(torch.int32)[160, 6] = -1
        t["i"].view(torch.int32)[160, 6] = -1
    state = torch.randn(5, d, generator=gen(16)).to(dev)
    state[0, 7] = float("nan")
    state[3, 8] = float("inf")
    h0 = state.clone()
    clean_h0 = h0.nan_to_num(0, 0, 0)
    carry, carry_c = (torch.empty(-(-sum(lens) // 64), d, device=dev) for _ in range(2))
    y = mamba_hip.gated_scan_packed(**t, cu_seqlens=cu(lens, dev), state=state, carry=carry)
    want = mamba_hip.gated_scan_packed(**clean, cu_seqlens=cu(lens, dev), state=clean_h0.clone(), carry=carry_c)
    bad = torch.zeros(sum(lens), d, dtype=torch.bool, device=dev)
    for row, c in ((150, 2), (500, 3), (2700, 4), (120, 5), (0, 7), (490, 8)) + (((160, 6),) if dtype == F32 else ()):
        s = max(s for s in starts if s <= row)
        bad[row:s + lens[starts.index(s)], c] = True
    assert torch.equal(torch.isfinite(y), ~bad)
    assert torch.equal(y[~bad], want[~bad])
    dy = torch.randn(sum(lens), d, generator=gen(17)).to(dtype).to(dev)
    got = mamba_hip.gated_scan_packed_bwd(dy, **t, cu_seqlens=cu(lens, dev), carry=carry, initial_state=h0)
    ref = mamba_hip.gated_scan_packed_bwd(dy, **clean, cu_seqlens=cu(lens, dev), carry=carry_c, initial_state=clean_h0)
    whole = torch.zeros_like(bad)  # a whole sequence's channel may be touched, nothing else
    for s, n in zip(starts, lens):
        whole[s:s + n] = bad[s:s + n].any(0)
    for key in ("dx", "dr", "di", "dz"):
        assert torch.equal(got[key][~whole], ref[key][~whole]), key
    touched = bad.any(0)
    assert torch.equal(got["dA"][~touched], ref["dA"][~touched]) and not torch.isfinite(got["dA"][touched]).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_outputs_in_place_and_rows_outside(dev, dtype):
    lens, d = LENS["mixed"], 70
    t = inputs(lens, d, dtype, dev, seed=18, pad=9)
    want = mamba_hip.gated_scan_packed(**t, cu_seqlens=cu(lens, dev))
    assert not want[-9:].any()
    out = torch.full((sum(lens) + 9, 2 * d), 7.0, dtype=dtype, device=dev)
    got = mamba_hip.gated_scan_packed(**t, cu_seqlens=cu(lens, dev), y=out[:, d:])
    assert torch.equal(got[:-9], want[:-9]) and bool((out[:, :d] == 7).all()) and bool((out[-9:] == 7).all())
    for key in ("x", "r", "i", "z"):
        t2 = {k: v.clone() for k, v in t.items()}
        got = mamba_hip.gated_scan_packed(**t2, cu_seqlens=cu(lens, dev), y=t2[key])
        assert got is t2[key] and torch.equal(got[:-9], want[:-9]), key
        assert got[-9:].isnan().all()


def test_sequences_without_a_slot(dev):
    lens, d = [5, 100, 70], 12
    t = inputs(lens, d, F32, dev, seed=19)
    state = torch.randn(4, d, generator=gen(20)).to(dev)
    before = state.clone()
    slots = torch.tensor([-1, 2, 4], dtype=torch.int32, device=dev)
    y = mamba_hip.gated_scan_packed(**t, cu_seqlens=cu(lens, dev), state=state, slots=slots)
    h0 = torch.zeros(3, d)
    h0[1] = before[2].cpu()
    ref = go.gated(lens, **t, h0=h0)
    k = roundings(lens, t)
    go.close(y, *ref["y"], k, "y")
    go.close(state[2], ref["hT"][0][1], ref["hT"][1][1], k, "state")
    assert torch.equal(state[[0, 1, 3]], before[[0, 1, 3]])


@pytest.mark.parametrize("b,d,dtype,z", [(1, 1, F32, True), (3, 257, BF16, True), (65, 1000, F32, False), (17, 2560, BF16, False),
                                         (300, 70, BF16, True), (2, 5120, F32, True)])
def test_step(dev, b, d, dtype, z):
    t = inputs([1] * b, d, dtype, dev, seed=21, z=z)
    slots = torch.randperm(b + 5, generator=gen(22))[:b].to(torch.int32)
    state = torch.randn(b + 5, d, generator=gen(23)).to(dev)
    before = state.clone()
    ref = go.gated([1] * b, **t, h0=state.cpu()[slots.long()])
    y = mamba_hip.gated_step_slots(**t, state=state, slots=slots.to(dev))
    k = roundings([1], t)
    go.close(y, *ref["y"], k, "y")
    go.close(state[slots.long()], *ref["hT"], k, "state")
    others = [i for i in range(b + 5) if i not in slots.tolist()]
    assert torch.equal(state[others], before[others])
    # the packed call on sequences of one token agrees with it bit for bit
    packed = before.clone()
    assert torch.equal(mamba_hip.gated_scan_packed(**t, cu_seqlens=cu([1] * b, dev), state=packed, slots=slots.to(dev)), y)
    assert torch.equal(packed, state)
    # slots out of range: zero rows, nothing kept
    slots[0] = b + 5
    state = before.clone()
    y2 = mamba_hip.gated_step_slots(**t, state=state, slots=slots.to(dev))
    assert not y2[0].any() and torch.equal(y2[1:], y[1:])
    assert torch.equal(state[others], before[others])
    # without slots: row s; into x itself
    state, x = before.clone(), t["x"].clone()
    y3 = mamba_hip.gated_step_slots(**{**t, "x": x}, state=state, slots=None, y=x)
    ref = go.gated([1] * b, **t, h0=before[:b])
    go.close(y3, *ref["y"], k, "y without slots")


def test_prefill_then_steps(dev):
    """A prompt in two segments and then token by token is the sequence in one call."""
    d, n = 33, 150
    t = inputs([n], d, F32, dev, seed=24)
    want_state = torch.zeros(1, d, device=dev)
    want = mamba_hip.gated_scan_packed(**t, cu_seqlens=cu([n], dev), state=want_state)
    state, rows = torch.zeros(1, d, device=dev), []
    for a, b in ((0, 70), (70, 140)):
        part = {k: v if k == "A" else v[a:b] for k, v in t.items()}
        rows.append(mamba_hip.gated_scan_packed(**part, cu_seqlens=cu([b - a], dev), state=state))
    for s in range(140, n):
        rows.append(mamba_hip.gated_step_slots(**{k: v if k == "A" else v[s:s + 1] for k, v in t.items()}, state=state, slots=None))
    ref = go.gated([n], **t)
    k = roundings([n], t)
    go.close(torch.cat(rows), *ref["y"], k, "segments")
    go.close(want, *ref["y"], k, "whole")
    go.close(state, *ref["hT"], k, "state")


def test_captured_and_replayed(dev):
    """Forward with a cache, and a training step, captured; replays with eager work between."""
    lens, d = LENS["groups"], 40
    t = inputs(lens, d, BF16, dev, seed=25)
    c = cu(lens, dev)
    state0 = torch.randn(len(lens), d, generator=gen(26)).to(dev)
    eager_state = state0.clone()
    eager = [mamba_hip.gated_scan_packed(**t, cu_seqlens=c, state=eager_state) for _ in range(3)]
    leaves = {k: v.detach().clone().requires_grad_() for k, v in t.items()}
    dy = torch.randn(sum(lens), d, generator=gen(27)).to(BF16).to(dev)

    def train():
        y, _ = mamba_hip.gated_scan_packed_autograd(**leaves, cu_seqlens=c)
        return torch.autograd.grad(y, list(leaves.values()), dy)

    want = [g.clone() for g in train()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
    torch.cuda.current_stream().wait_stream(side)
    state = state0.clone()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y = mamba_hip.gated_scan_packed(**t, cu_seqlens=c, state=state)
    with torch.cuda.graph(g2):
        grads = train()
    for rep in range(3):
        g1.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager[rep]), rep
        mamba_hip.gated_scan_packed(**t, cu_seqlens=c)
        g2.replay()
        torch.cuda.synchronize()
        for a, b in zip(grads, want):
            assert torch.equal(a, b), rep
    assert torch.equal(state, eager_state)


def test_rows_that_are_one(dev):
    """A row that all tokens share (stride 0) is read as its copies are; so is every second row."""
    lens, d = LENS["mixed"], 70
    t = inputs(lens, d, F32, dev, seed=31)
    n, c = sum(lens), cu(lens, dev)
    one = {**t, "r": t["r"][:1].expand(n, d), "i": torch.randn(2 * n, d, generator=gen(32)).to(dev)[::2]}
    copies = {k: v.clone(memory_format=torch.contiguous_format) for k, v in one.items()}
    carry, carry2 = (torch.zeros(-(-n // 64), d, device=dev) for _ in range(2))
    assert torch.equal(mamba_hip.gated_scan_packed(**one, cu_seqlens=c, carry=carry), mamba_hip.gated_scan_packed(**copies, cu_seqlens=c, carry=carry2))
    dy = torch.randn(1, d, generator=gen(33)).to(dev).expand(n, d)
    a = mamba_hip.gated_scan_packed_bwd(dy, **one, cu_seqlens=c, carry=carry)
    b = mamba_hip.gated_scan_packed_bwd(dy.contiguous(), **copies, cu_seqlens=c, carry=carry2)
    assert all(torch.equal(a[k], b[k]) for k in ("dx", "dr", "di", "dz", "dA"))


def test_two_streams_at_once(dev):
    """Calls that run side by side share nothing."""
    lens, d = LENS["groups"], 200
    ts = [inputs(lens, d, F32, dev, seed=30 + k) for k in range(2)]
    c = cu(lens, dev)
    want = [mamba_hip.gated_scan_packed(**t, cu_seqlens=c) for t in ts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(mamba_hip.gated_scan_packed(**ts[k], cu_seqlens=c))
    torch.cuda.synchronize()
    for k in range(2):
        for y in got[k]:
            assert torch.equal(y, want[k])


def test_no_rows(dev):
    e = torch.empty(0, 5, device=dev)
    A, c = -torch.ones(5, device=dev), cu([0, 0], dev)
    state = torch.randn(2, 5, generator=gen(28)).to(dev)
    before = state.clone()
    assert mamba_hip.gated_scan_packed(e, e, e, A, c, state=state).shape == (0, 5)
    assert torch.equal(state, before)
    got = mamba_hip.gated_scan_packed_bwd(e, e, e, e, A, c, torch.empty(0, 5, device=dev), initial_state=state, d_final_state=state)
    assert not got["dA"].any() and torch.equal(got["d_initial_state"], state) and got["dx"].shape == (0, 5)
    assert mamba_hip.gated_step_slots(e, e, e, A, state, torch.empty(0, dtype=torch.int32, device=dev)).shape == (0, 5)
