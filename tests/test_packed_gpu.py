"""The packed convolution and selective scan, their gradients and the slot steps
against plain 64-bit forms (packed_oracle), where they can go wrong: empty and
one-row sequences, sequences across chunk borders, odd widths, padded states,
strided rows, padding rows that hold NaN, slots out of range."""

import pytest
import torch

import mamba_hip
import packed_oracle as po

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

LENS = {
    "one": [1],
    "short": [7],
    "mixed": [0, 1, 130, 0, 63, 200, 5, 0],
    "borders": [64, 64, 128, 1, 127],
    "long": [700],
    "tokens": [1] * 70,
    "thousands": [30000, 1, 20011],
    "many chunks": [6000, 1, 0, 199],
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


def scan_inputs(lens, d, n, dtype, dev, seed=0, pad=0, full=True):
    g, rows = gen(seed), sum(lens) + pad
    t = dict(u=strided(g, rows, d, dtype, dev), delta=strided(g, rows, d, dtype, dev),
             A=(-torch.exp(torch.rand(d, n, generator=g) * 2.5)).to(dev),
             B=strided(g, rows, n, dtype, dev, 5, 0), C=strided(g, rows, n, dtype, dev, 0, 3))
    if full:
        t.update(D=torch.randn(d, generator=g).to(dev), z=strided(g, rows, d, dtype, dev),
                 delta_bias=(torch.randn(d, generator=g) - 3).to(dev))
    else:
        t["delta"] = t["delta"].abs() * 0.1
    if pad:
        for k in ("u", "delta", "B", "C", "z"):
            if k in t:
                t[k][-pad:] = float("nan")
    return t


def oracle_args(t, full):
    return dict(u=t["u"], delta=t["delta"], A=t["A"], B=t["B"], C=t["C"], D=t.get("D"), z=t.get("z"), bias=t.get("delta_bias"), sp=full)


def roundings(lens):
    return 40 + 4 * max(lens + [0])


CASES = [("one", 1, 1, F32, 0, True), ("short", 5, 16, BF16, 2, False), ("mixed", 70, 16, F32, 3, True),
         ("mixed", 64, 16, BF16, 0, True), ("borders", 37, 20, F32, 0, True), ("long", 65, 5, BF16, 1, False),
         ("mixed", 33, 32, BF16, 0, True), ("borders", 18, 64, F32, 2, True), ("short", 9, 33, F32, 0, True),
         ("tokens", 40, 16, F32, 0, True), ("mixed", 130, 8, BF16, 3, True), ("many chunks", 8, 5, F32, 0, True)]


@pytest.mark.parametrize("name,d,n,dtype,pad,full", CASES)
def test_scan_forward(dev, name, d, n, dtype, pad, full):
    lens = LENS[name]
    t = scan_inputs(lens, d, n, dtype, dev, pad=pad, full=full)
    slots = torch.randperm(len(lens) + 3, generator=gen(1))[:len(lens)].to(torch.int32)
    state = torch.randn(len(lens) + 3, d, n, generator=gen(2)).to(dev)
    ref = po.scan(lens, h0=state.cpu()[slots.long()], **oracle_args(t, full))
    before = state.clone()
    y = mamba_hip.mamba1_scan_packed(**t, cu_seqlens=cu(lens, dev), delta_softplus=full, state=state, slots=slots.to(dev))
    po.close(y, *ref["y"], roundings(lens), "y")
    po.close(state[slots.long()], *ref["hT"], roundings(lens), "state")
    others = [i for i in range(len(lens) + 3) if i not in slots.tolist()]
    assert torch.equal(state[others], before[others])
    # without a state: from zero, nothing kept; the bound on the lengths changes nothing but the schedule
    ref = po.scan(lens, **oracle_args(t, full))
    for most in (0, max(lens)):
        y = mamba_hip.mamba1_scan_packed(**t, cu_seqlens=cu(lens, dev), delta_softplus=full, max_seqlen=most)
        po.close(y, *ref["y"], roundings(lens), "y from zero")


@pytest.mark.parametrize("name,d,n,dtype,pad,full", CASES)
def test_scan_backward(dev, name, d, n, dtype, pad, full):
    lens = LENS[name]
    t = scan_inputs(lens, d, n, dtype, dev, seed=3, pad=pad, full=full)
    g = gen(4)
    h0, dhT = (torch.randn(len(lens), d, n, generator=g).to(dev) for _ in range(2))
    dy = strided(g, sum(lens) + pad, d, dtype, dev)
    if pad:
        dy[-pad:] = float("nan")
    for start in (None, h0):
        back = None if start is None else dhT
        ref = po.scan(lens, h0=start, dy=dy, dhT=back, **oracle_args(t, full))
        got = mamba_hip.mamba1_scan_packed_bwd(dy, **t, cu_seqlens=cu(lens, dev), delta_softplus=full, initial_state=start,
                                               d_final_state=back)
        k = roundings(lens)
        for name_ in ("du", "ddelta", "dB", "dC"):
            po.close(got[name_], *ref[name_], 2 * k, name_)
        # sums over the rows besides: in chunks and then over the chunks
        more = 2 * k + sum(lens)
        po.close(got["dA"], *ref["dA"], more, "dA")
        if full:
            po.close(got["dz"], *ref["dz"], 2 * k, "dz")
            po.close(got["dD"], *ref["dD"], more, "dD")
            po.close(got["d_delta_bias"], *ref["dbias"], more, "d_delta_bias")
        else:
            assert got["dz"] is None and got["dD"] is None and got["d_delta_bias"] is None
        if start is None:
            assert got["d_initial_state"] is None
        else:
            po.close(got["d_initial_state"], *ref["dh0"], 2 * k, "d_initial_state")
    again = mamba_hip.mamba1_scan_packed_bwd(dy, **t, cu_seqlens=cu(lens, dev), delta_softplus=full, initial_state=h0,
                                             d_final_state=dhT)
    for key, v in got.items():
        assert v is None or torch.equal(v, again[key]), key


def test_scan_gradient_by_differences(dev):
    """The gradient along a direction against the difference quotient of the 64-bit form."""
    lens = [3, 70, 0, 20]
    t = scan_inputs(lens, 6, 7, F32, dev, seed=5)
    dy = torch.randn(sum(lens), 6, generator=gen(6)).to(dev)
    got = mamba_hip.mamba1_scan_packed_bwd(dy, **t, cu_seqlens=cu(lens, dev), delta_softplus=True)
    names = dict(u="du", delta="ddelta", A="dA", B="dB", C="dC", D="dD", z="dz", delta_bias="d_delta_bias")
    for k, gk in names.items():
        v = torch.randn(t[k].shape, generator=gen(7), dtype=torch.float64)
        step = 1e-5

        def objective(sign):
            moved = {key: po.d(x) for key, x in t.items()}
            moved[k] = moved[k] + sign * step * v
            return float((po.scan(lens, **oracle_args(moved, True))["y"][0] * po.d(dy)).sum())

        quotient = (objective(1) - objective(-1)) / (2 * step)
        along = float((po.d(got[gk]) * v).sum())
        # the quotient is off by step^2 of third derivatives, the gradient by f32 roundings
        assert abs(along - quotient) <= 1e-4 * (abs(quotient) + float((po.d(got[gk]).abs() * v.abs()).sum())), (k, along, quotient)


@pytest.mark.parametrize("name", ["mixed", "long"])
def test_scan_autograd(dev, name):
    lens, d, n = LENS[name], 24, 16
    t = scan_inputs(lens, d, n, F32, dev, seed=8)
    h0 = torch.randn(len(lens), d, n, generator=gen(9)).to(dev)
    leaves = {k: v.detach().clone().requires_grad_() for k, v in t.items()}
    h = h0.clone().requires_grad_()
    y, hT = mamba_hip.mamba1_scan_packed_autograd(**leaves, cu_seqlens=cu(lens, dev), delta_softplus=True, initial_state=h)
    (y.sum() + 2 * hT.sum()).backward()  # expanded gradients
    ref = mamba_hip.mamba1_scan_packed_bwd(torch.ones_like(y), **t, cu_seqlens=cu(lens, dev), delta_softplus=True, initial_state=h0,
                                           d_final_state=torch.full_like(h0, 2.0))
    names = dict(u="du", delta="ddelta", A="dA", B="dB", C="dC", D="dD", z="dz", delta_bias="d_delta_bias")
    for k, gk in names.items():
        assert torch.equal(leaves[k].grad, ref[gk]), k
    assert torch.equal(h.grad, ref["d_initial_state"])
    # only one of the outputs used
    y, hT = mamba_hip.mamba1_scan_packed_autograd(**leaves, cu_seqlens=cu(lens, dev), delta_softplus=True)
    gu, = torch.autograd.grad(hT.sum(), [leaves["u"]])
    assert torch.isfinite(gu).all() and gu.any()


def test_scan_in_parts_equals_whole(dev):
    """A sequence run in pieces through its slot ends where the whole one does."""
    d, n = 48, 16
    t = scan_inputs([300], d, n, F32, dev, seed=10)
    whole = torch.zeros(2, d, n, device=dev)
    y = mamba_hip.mamba1_scan_packed(**t, cu_seqlens=cu([300], dev), delta_softplus=True, state=whole, slots=torch.ones(1, dtype=torch.int32, device=dev))
    state, parts, at = torch.zeros(2, d, n, device=dev), [], 0
    slots = torch.ones(1, dtype=torch.int32, device=dev)
    for step in (100, 1, 63, 136):
        piece = {k: (v[at:at + step] if k in ("u", "delta", "B", "C", "z") else v) for k, v in t.items()}
        parts.append(mamba_hip.mamba1_scan_packed(**piece, cu_seqlens=cu([step], dev), delta_softplus=True, state=state, slots=slots))
        at += step
    ref = po.scan([300], **oracle_args(t, True))
    po.close(torch.cat(parts), *ref["y"], roundings([300]), "y in parts")
    po.close(state[1:], *ref["hT"], roundings([300]), "state in parts")
    po.close(y, *ref["y"], roundings([300]), "y")
    assert not state[0].any()


def test_scan_nan_stays_in_its_sequence(dev):
    lens, d, n = [90, 40, 200], 20, 16
    t = scan_inputs(lens, d, n, F32, dev, seed=11)
    clean = mamba_hip.mamba1_scan_packed(**t, cu_seqlens=cu(lens, dev), delta_softplus=True)
    t["u"][100] = float("nan")
    t["z"][101] = float("inf")
    y = mamba_hip.mamba1_scan_packed(**t, cu_seqlens=cu(lens, dev), delta_softplus=True)
    assert torch.equal(y[:100], clean[:100]) and torch.equal(y[130:], clean[130:]) and y[100:130].isnan().all()
    dy = torch.ones_like(y)
    g = mamba_hip.mamba1_scan_packed_bwd(dy, **t, cu_seqlens=cu(lens, dev), delta_softplus=True)
    for k in ("du", "ddelta", "dz", "dB", "dC"):
        assert torch.isfinite(g[k][:90]).all() and torch.isfinite(g[k][130:]).all(), k


def test_rows_outside_and_slots_out_of_range(dev):
    """Padding rows of a given output keep what they hold; a slot out of range is no state;
    wrong offsets touch nothing out of the tensors."""
    lens, d, n, pad = [5, 80], 12, 16, 9
    t = scan_inputs(lens, d, n, F32, dev, seed=12, pad=pad)
    y = torch.full((sum(lens) + pad, d), 7.0, device=dev)
    state = torch.randn(3, d, n, generator=gen(1)).to(dev)
    before = state.clone()
    slots = torch.tensor([-1, 3], dtype=torch.int32, device=dev)
    mamba_hip.mamba1_scan_packed(**t, cu_seqlens=cu(lens, dev), delta_softplus=True, state=state, slots=slots, y=y)
    assert torch.equal(state, before) and (y[-pad:] == 7).all()
    po.close(y[:-pad], po.scan(lens, **oracle_args(t, True))["y"][0][:-pad], po.scan(lens, **oracle_args(t, True))["y"][1][:-pad],
             roundings(lens), "y")
    x, w = t["u"], torch.randn(d, 4, generator=gen(2)).to(dev)
    out = torch.full_like(y, 7.0)
    win = torch.randn(3, d, 4, generator=gen(3)).to(dev)
    keep = win.clone()
    mamba_hip.conv1d_packed(x, w, cu(lens, dev), state=win, slots=slots, out=out)
    assert torch.equal(win, keep) and (out[-pad:] == 7).all()
    for wrong in ([0, 300, 20, 94], [50, 10, -7, 2 ** 31 - 1], [94, 94, 0, 0]):
        c = torch.tensor(wrong, dtype=torch.int32, device=dev)
        mamba_hip.mamba1_scan_packed(**t, cu_seqlens=c, delta_softplus=True, state=state.clone())
        mamba_hip.mamba1_scan_packed_bwd(y, **t, cu_seqlens=c, delta_softplus=True, initial_state=state)
        mamba_hip.conv1d_packed(x, w, c, state=win.clone())
        mamba_hip.conv1d_packed_bwd(y, x, w, c)
    torch.cuda.synchronize()


def test_scan_of_whole_sequences(dev):
    """A known bound on the lengths: a workgroup takes whole sequences and nothing is carried.
    Rows before, between and behind the sequences, a wrong bound, and slots."""
    lens, d, n = [40, 0, 96, 1, 64, 30], 30, 16
    rows = 5 + sum(lens) + 7
    t = scan_inputs([rows], d, n, BF16, dev, seed=23)
    starts = [5]
    for k in lens:
        starts.append(starts[-1] + k)
    c = torch.tensor(starts, dtype=torch.int32, device=dev)
    slots = torch.tensor([3, 6, 0, 1, 5, 2], dtype=torch.int32, device=dev)
    state = torch.randn(7, d, n, generator=gen(24)).to(dev)
    inner = {k: (v[5:] if k in ("u", "delta", "B", "C", "z") else v) for k, v in t.items()}
    ref = po.scan(lens, h0=state.cpu()[slots.long().cpu()], **oracle_args(inner, True))
    for most in (96, 1, 0):  # known, wrong (the schedule only), unknown
        h, y = state.clone(), torch.full((rows, d), 7.0, dtype=BF16, device=dev)
        mamba_hip.mamba1_scan_packed(**t, cu_seqlens=c, delta_softplus=True, state=h, slots=slots, max_seqlen=most, y=y)
        po.close(y[5:-7], ref["y"][0][:-7], ref["y"][1][:-7], roundings(lens), "y")
        assert (y[:5] == 7).all() and (y[-7:] == 7).all()
        po.close(h[slots.long()], *ref["hT"], roundings(lens), "state")
        assert torch.equal(h[4], state[4])
        y = mamba_hip.mamba1_scan_packed(**t, cu_seqlens=c, delta_softplus=True, max_seqlen=most)
        assert not y[:5].any() and not y[-7:].any() and y[5:-7].any()


CONV = [("one", 3, 4, F32, 0, True), ("mixed", 130, 4, BF16, 3, True), ("borders", 600, 3, F32, 0, True),
        ("long", 77, 2, BF16, 5, False), ("mixed", 9, 1, F32, 0, True), ("tokens", 260, 4, F32, 0, True),
        ("mixed", 70, 7, F32, 2, True), ("short", 5, 64, BF16, 0, True),
        ("mixed", 129, 8, F32, 0, True), ("borders", 131, 5, BF16, 3, True), ("mixed", 2, 6, F32, 2, False), ("long", 5, 4, BF16, 0, True),
        ("tokens", 33, 9, F32, 0, True), ("thousands", 5, 4, F32, 7, True)]


@pytest.mark.parametrize("name,c,k,dtype,pad,act", CONV)
def test_conv(dev, name, c, k, dtype, pad, act):
    lens, g = LENS[name], gen(13)
    rows = sum(lens) + pad
    x, dout = strided(g, rows, c, dtype, dev), strided(g, rows, c, dtype, dev)
    if pad:
        x[-pad:], dout[-pad:] = float("nan"), float("nan")
    w = (torch.randn(c, k, generator=g) / k ** 0.5).to(dev)
    bias = torch.randn(c, generator=g).to(dev) if act else None
    # k products and sums, the sigmoid's exp and reciprocal, a product
    few = k + 8
    window = torch.randn(len(lens) + 2, c, k, generator=g).to(dev)
    slots = torch.randperm(len(lens) + 2, generator=g)[:len(lens)].to(torch.int32)
    ref = po.conv(lens, x, w, bias, act, window.cpu()[slots.long()])
    y = mamba_hip.conv1d_packed(x, w, cu(lens, dev), bias, act, window, slots.to(dev))
    po.close(y[:rows - pad], ref["y"][0][:rows - pad], ref["y"][1][:rows - pad], few, "y")
    assert not y[rows - pad:].any()
    assert torch.equal(po.d(window[slots.long()]), ref["window"][0])
    ref = po.conv(lens, x, w, bias, act, None, dout)
    y = mamba_hip.conv1d_packed_autograd(x, w, cu(lens, dev), bias, act)
    po.close(y[:rows - pad], ref["y"][0][:rows - pad], ref["y"][1][:rows - pad], few, "y from zero")
    got = mamba_hip.conv1d_packed_bwd(dout, x, w, cu(lens, dev), bias, act)
    po.close(got["dx"][:rows - pad], ref["dx"][0][:rows - pad], ref["dx"][1][:rows - pad], 2 * few, "dx")
    assert not got["dx"][rows - pad:].any()
    po.close(got["dw"], *ref["dw"], 2 * few + rows, "dw")
    if act:
        po.close(got["dbias"], *ref["dbias"], 2 * few + rows, "dbias")
    again = mamba_hip.conv1d_packed_bwd(dout, x, w, cu(lens, dev), bias, act)
    assert all(v is None or torch.equal(v, again[key]) for key, v in got.items())


def test_conv_autograd(dev):
    lens, g = LENS["mixed"], gen(14)
    x = strided(g, sum(lens), 40, BF16, dev).detach().requires_grad_()
    w = torch.randn(40, 4, generator=g).to(dev).requires_grad_()
    b = torch.randn(40, generator=g).to(dev).requires_grad_()
    y = mamba_hip.conv1d_packed_autograd(x, w, cu(lens, dev), b)
    y.sum().backward()
    ref = mamba_hip.conv1d_packed_bwd(torch.ones_like(y), x.detach(), w.detach(), cu(lens, dev), b.detach())
    assert torch.equal(x.grad, ref["dx"]) and torch.equal(w.grad, ref["dw"]) and torch.equal(b.grad, ref["dbias"])


@pytest.mark.parametrize("b,d,n,k,dtype,full", [(1, 1, 1, 1, F32, True), (5, 70, 16, 4, BF16, True), (33, 130, 20, 3, F32, False),
                                                (2, 300, 64, 4, BF16, True), (3, 40, 100, 2, F32, True), (7, 256, 16, 4, F32, True),
                                                (4, 200, 12, 4, BF16, True), (2, 1030, 1, 3, F32, True), (3, 5, 1000, 4, F32, False),
                                                (2, 700, 3, 5, F32, True), (3, 90, 8, 7, BF16, True), (2, 33, 16, 8, F32, True), (2, 33, 16, 9, F32, True)])
def test_steps(dev, b, d, n, k, dtype, full):
    """One token per slot: the packed forms of one-row sequences are the same function."""
    g, lens = gen(15), [1] * b
    t = scan_inputs(lens, d, n, dtype, dev, seed=16, full=full)
    state, window = torch.randn(b + 4, d, n, generator=g).to(dev), torch.randn(b + 4, d, k, generator=g).to(dev)
    slots = torch.randperm(b + 4, generator=g)[:b].to(torch.int32)
    w, bias = torch.randn(d, k, generator=g).to(dev), torch.randn(d, generator=g).to(dev)
    ref = po.scan(lens, h0=state.cpu()[slots.long()], **oracle_args(t, full))
    before = state.clone()
    y = mamba_hip.scan_step_slots(t["u"], t["delta"], t["A"], t["B"], t["C"], state, slots.to(dev), t.get("D"), t.get("z"),
                                  t.get("delta_bias"), full)
    po.close(y, *ref["y"], 44 + n, "y")
    po.close(state[slots.long()], *ref["hT"], 44, "state")
    others = [i for i in range(b + 4) if i not in slots.tolist()]
    assert torch.equal(state[others], before[others])
    ref = po.conv(lens, t["u"], w, bias, True, window.cpu()[slots.long()])
    out = mamba_hip.conv1d_step_slots(t["u"], window, slots.to(dev), w, bias)
    po.close(out, *ref["y"], k + 8, "conv")
    assert torch.equal(po.d(window[slots.long()]), ref["window"][0])


def test_steps_without_a_slot(dev):
    t = scan_inputs([1] * 4, 20, 16, F32, dev, seed=17)
    state, window = torch.randn(4, 20, 16).to(dev), torch.randn(4, 20, 4).to(dev)
    w = torch.randn(20, 4).to(dev)
    slots = torch.tensor([2, -1, 9, 0], dtype=torch.int32, device=dev)
    s0, w0 = state.clone(), window.clone()
    y = mamba_hip.scan_step_slots(t["u"], t["delta"], t["A"], t["B"], t["C"], state, slots, delta_softplus=True)
    out = mamba_hip.conv1d_step_slots(t["u"], window, slots, w)
    assert not y[1:3].any() and not out[1:3].any() and y[0].any() and out[3].any()
    assert torch.equal(state[[1, 3]], s0[[1, 3]]) and torch.equal(window[[1, 3]], w0[[1, 3]])


def test_nothing_to_do(dev):
    """No rows, no sequences, no tokens."""
    e = lambda *s: torch.empty(*s, device=dev)  # noqa: E731
    A = -torch.ones(6, 16, device=dev)
    for rows, c in ((0, [0]), (0, [0, 0, 0]), (4, [0]), (4, [0, 0])):
        offsets = torch.tensor(c, dtype=torch.int32, device=dev)
        y = mamba_hip.mamba1_scan_packed(e(rows, 6), e(rows, 6), A, e(rows, 16), e(rows, 16), offsets)
        assert y.shape == (rows, 6) and not y.any()
        g = mamba_hip.mamba1_scan_packed_bwd(e(rows, 6), e(rows, 6), e(rows, 6), A, e(rows, 16), e(rows, 16), offsets,
                                             initial_state=torch.ones(len(c) - 1, 6, 16, device=dev))
        assert not any(g[k].any() for k in ("du", "ddelta", "dA", "dB", "dC", "d_initial_state"))
        assert not mamba_hip.conv1d_packed(e(rows, 6), e(6, 4), offsets).any()
        g = mamba_hip.conv1d_packed_bwd(e(rows, 6), e(rows, 6), e(6, 4), offsets, e(6))
        assert not any(g[k].any() for k in ("dx", "dw", "dbias"))
    none = torch.empty(0, dtype=torch.int32, device=dev)
    assert mamba_hip.scan_step_slots(e(0, 6), e(0, 6), A, e(0, 16), e(0, 16), e(2, 6, 16), none).shape == (0, 6)
    assert mamba_hip.conv1d_step_slots(e(0, 6), e(2, 6, 4), none, e(6, 4)).shape == (0, 6)


def test_outputs_in_place(dev):
    """y over u, delta or z, and beside them in one tensor."""
    lens, d, n = LENS["mixed"], 40, 16
    t = scan_inputs(lens, d, n, BF16, dev, seed=25)
    want = mamba_hip.mamba1_scan_packed(**t, cu_seqlens=cu(lens, dev), delta_softplus=True)
    for k in ("u", "delta", "z"):
        mine = {key: v.clone() for key, v in t.items()}
        y = mamba_hip.mamba1_scan_packed(**mine, cu_seqlens=cu(lens, dev), delta_softplus=True, y=mine[k])
        assert y is mine[k] and torch.equal(y, want), k
    both = torch.zeros(sum(lens), 2 * d, dtype=BF16, device=dev)
    both[:, :d] = t["u"]
    mamba_hip.mamba1_scan_packed(**{**t, "u": both[:, :d]}, cu_seqlens=cu(lens, dev), delta_softplus=True, y=both[:, d:])
    assert torch.equal(both[:, d:], want) and torch.equal(both[:, :d], t["u"])


def test_many_empty_sequences(dev):
    """Empty ones in the middle are passed over, and end in what they start from."""
    lens = [70] + [0] * 5000 + [70]
    t = scan_inputs([140], 16, 16, F32, dev, seed=26)
    c = cu(lens, dev)
    state = torch.randn(len(lens), 16, 16, generator=gen(27)).to(dev)
    before = state.clone()
    y = mamba_hip.mamba1_scan_packed(**t, cu_seqlens=c, delta_softplus=True, state=state)
    ends = [0, len(lens) - 1]
    ref = po.scan([70, 70], h0=before.cpu()[ends], **oracle_args(t, True))
    po.close(y, *ref["y"], roundings([70]), "y")
    po.close(state[ends], *ref["hT"], roundings([70]), "state")
    assert torch.equal(state[1:-1], before[1:-1])
    dy, dhT = torch.ones_like(y), torch.randn(len(lens), 16, 16, generator=gen(28)).to(dev)
    g = mamba_hip.mamba1_scan_packed_bwd(dy, **t, cu_seqlens=c, delta_softplus=True, initial_state=before, d_final_state=dhT)
    assert torch.equal(g["d_initial_state"][1:-1], dhT[1:-1])
    ref = po.scan([70, 70], h0=before.cpu()[ends], dy=dy, dhT=dhT.cpu()[ends], **oracle_args(t, True))
    po.close(g["d_initial_state"][ends], *ref["dh0"], 2 * roundings([70]), "dh0")
    w = torch.randn(16, 4, generator=gen(29)).to(dev)
    x = t["u"]
    po.close(mamba_hip.conv1d_packed(x, w, c), *po.conv([70, 70], x, w)["y"], 12, "conv")


def test_twice_differentiated(dev):
    """A second derivative is refused, not wrong."""
    lens = [9, 30]
    t = {k: v.detach().requires_grad_() for k, v in scan_inputs(lens, 8, 16, F32, dev, seed=30).items()}
    y, _ = mamba_hip.mamba1_scan_packed_autograd(**t, cu_seqlens=cu(lens, dev), delta_softplus=True)
    dy = torch.ones_like(y).requires_grad_()
    g, = torch.autograd.grad(y, [t["u"]], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_graph_and_streams(dev):
    """Captured and replayed on other values, with eager calls on another stream between."""
    lens, d, n = [40, 200, 1], 64, 16
    t = scan_inputs(lens, d, n, F32, dev, seed=18)
    t = {k: v.contiguous() for k, v in t.items()}
    other = scan_inputs(lens, d, n, F32, dev, seed=19)
    c, dy = cu(lens, dev), torch.randn(sum(lens), d, generator=gen(20)).to(dev)
    w, bias = torch.randn(d, 4, generator=gen(21)).to(dev), torch.randn(d, generator=gen(22)).to(dev)
    state = torch.zeros(3, d, n, device=dev)

    def work():
        x = mamba_hip.conv1d_packed(t["u"], w, c, bias)
        y = mamba_hip.mamba1_scan_packed(x, t["delta"], t["A"], t["B"], t["C"], c, t["D"], t["z"], t["delta_bias"], True, state)
        g = mamba_hip.mamba1_scan_packed_bwd(dy, x, t["delta"], t["A"], t["B"], t["C"], c, t["D"], t["z"], t["delta_bias"], True)
        gc = mamba_hip.conv1d_packed_bwd(g["du"], t["u"], w, c, bias)
        return [y, g["dA"], g["dB"], g["d_delta_bias"], gc["dx"], gc["dw"]]

    work()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        captured = work()
    for k in range(3):
        for key in t:
            t[key].copy_(other[key] * (1 + 0.1 * k))
        state.fill_(0.5 * k)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in captured] + [state.clone()]
        state.fill_(0.5 * k)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = work() + [state.clone()]
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_slots_far_into_a_cache(dev):
    """Slots whose states lie behind 2^31 elements, as in a small cache."""
    d, n, k, far, wide = 5120, 16, 4, 26999, 104999
    t = scan_inputs([40, 3], d, n, BF16, dev, seed=31)
    c, w = cu([40, 3], dev), torch.randn(d, k, generator=gen(32)).to(dev)
    near, there = torch.tensor([1, 0], dtype=torch.int32, device=dev), torch.tensor([far, 2], dtype=torch.int32, device=dev)
    small = torch.randn(2, d, n, generator=gen(33)).to(dev)
    state = torch.empty(far + 1, d, n, device=dev)
    state[there.long()] = small[near.long()]
    assert state[far].storage_offset() > 2 ** 31
    for call in (lambda h, slots: mamba_hip.mamba1_scan_packed(**t, cu_seqlens=c, delta_softplus=True, state=h, slots=slots),
                 lambda h, slots: mamba_hip.mamba1_scan_packed(**t, cu_seqlens=c, delta_softplus=True, state=h, slots=slots, max_seqlen=40),
                 lambda h, slots: mamba_hip.scan_step_slots(**{key: v[:2] if key in ("u", "delta", "B", "C", "z") else v for key, v in t.items()},
                                                            state=h, slots=slots, delta_softplus=True)):
        assert torch.equal(call(state, there), call(small, near))
        assert torch.equal(state[there.long()], small[near.long()])
    del state
    there[0] = wide
    small = torch.randn(2, d, k, generator=gen(34)).to(dev)
    window = torch.empty(wide + 1, d, k, device=dev)
    window[there.long()] = small[near.long()]
    assert window[wide].storage_offset() > 2 ** 31
    assert torch.equal(mamba_hip.conv1d_packed(t["u"], w, c, state=window, slots=there),
                       mamba_hip.conv1d_packed(t["u"], w, c, state=small, slots=near))
    assert torch.equal(mamba_hip.conv1d_step_slots(t["u"][:2], window, there, w), mamba_hip.conv1d_step_slots(t["u"][:2], small, near, w))
    assert torch.equal(window[there.long()], small[near.long()])


def test_rows_far_apart(dev):
    """Rows behind 2^31 elements, read and written."""
    rows, d, n, pitch = 70, 40, 16, 2 ** 25 - 8
    t = scan_inputs([rows], d, n, BF16, dev, seed=35)
    base = torch.empty(rows * pitch, dtype=BF16, device=dev)
    at = 0

    def apart(v):
        nonlocal at
        out = base.as_strided((rows, v.shape[1]), (pitch, 1), at)
        at += v.shape[1] + 3
        return out.copy_(v)
    far = {k: apart(v) if k in ("u", "delta", "B", "C", "z") else v for k, v in t.items()}
    c, y, out = cu([30, 40], dev), apart(t["u"]), apart(t["u"])
    assert y[-1].storage_offset() > 2 ** 31
    kw = dict(cu_seqlens=c, delta_softplus=True)
    assert mamba_hip.mamba1_scan_packed(**far, **kw, y=y) is y
    want = mamba_hip.mamba1_scan_packed(**t, **kw)
    assert torch.equal(y, want)
    a, b = mamba_hip.mamba1_scan_packed_bwd(y, **far, **kw), mamba_hip.mamba1_scan_packed_bwd(want, **t, **kw)
    assert all(v is None or torch.equal(v, b[k]) for k, v in a.items())
    w = torch.randn(d, 4, generator=gen(36)).to(dev)
    assert torch.equal(mamba_hip.conv1d_packed(far["u"], w, c, out=out), mamba_hip.conv1d_packed(t["u"], w, c))
    a, b = mamba_hip.conv1d_packed_bwd(y, far["u"], w, c), mamba_hip.conv1d_packed_bwd(want, t["u"], w, c)
    assert all(v is None or torch.equal(v, b[k]) for k, v in a.items())
    scale, stats = torch.randn(d, generator=gen(37)).to(dev), [tuple(torch.empty(rows, device=dev) for _ in range(2)) for _ in range(2)]
    assert torch.equal(mamba_hip.layer_norm(far["u"], scale, out=out, stats=stats[0]), mamba_hip.layer_norm(t["u"], scale, stats=stats[1]))
    a, b = mamba_hip.layer_norm_bwd(y, far["u"], scale, *stats[0]), mamba_hip.layer_norm_bwd(want, t["u"], scale, *stats[1])
    assert all(torch.equal(v, b[k]) for k, v in a.items())
    rng = torch.tensor([3, 4], device=dev)
    assert torch.equal(mamba_hip.dropout(far["u"], 0.4, rng, residual=far["z"], out=out), mamba_hip.dropout(t["u"], 0.4, rng, residual=t["z"]))
