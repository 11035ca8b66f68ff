"""Sequences of hundreds of thousands of rows: the recurrence and its gradients over thousands of
tiles, against a scan by doubling in 64 bits.

Bounds: a row multiplies what it takes over by its decay and adds its term, in 4 + |w| (6 + 2 |r|)
roundings of 2^-23 (w = A s(r): the decay's own), so the error obeys the recurrence itself, e_t = a_t
e_{t-1} + that many roundings of the sum of the absolute values m_t; what is around it (weights,
gates, their slopes) has at most 40 + 4 (|r| + |i| + |z|) roundings."""

import pytest
import torch

import mamba_hip
from packed_oracle import half_step

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def scan(a, b, first, back=False):
    """h_t = a_t h_{t-1} + b_t (from 0 at a sequence's first row), or the same from the end."""
    P, H = torch.where(first[:, None], torch.zeros_like(a), a), b.clone()
    if back:  # h_t = b_t + a_{t+1} h_{t+1}
        P, H = torch.cat([P[1:], torch.zeros_like(P[:1])]).flip(0), H.flip(0)
    n, d = len(P), 1
    while d < n:
        H = torch.cat([H[:d], H[d:] + P[d:] * H[:-d]])
        P = torch.cat([P[:d], P[d:] * P[:-d]])
        d *= 2
    return H.flip(0) if back else H


def close(got, ref, err, what):
    tol = half_step(got.dtype) * ref.abs() * (1 + 2 ** -8) + err + 1e-37
    off = (got.double() - ref).abs()
    assert bool((off <= tol).all()), (what, float((off / tol).max()))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long(dev, dtype):
    lens, d = [100, 200001, 0, 1, 70000], 5
    n = sum(lens)
    g = torch.Generator(device=dev).manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x, r, i, z, dy = (mk(n, d).to(dtype) for _ in range(5))
    A = -torch.tensor([0.0005, 0.004, 0.03, 0.2, 2.0], device=dev)  # states that last from one row to thousands
    ends = torch.tensor(lens).cumsum(0).tolist()
    cu = torch.tensor([0] + ends, dtype=torch.int32, device=dev)
    state, carry = torch.zeros(len(lens), d, device=dev), torch.empty(-(-n // 64), d, device=dev)
    y = mamba_hip.gated_scan_packed(x, r, i, A, cu, z, state=state, carry=carry)
    grads = mamba_hip.gated_scan_packed_bwd(dy, x, r, i, A, cu, carry, z)
    first = torch.zeros(n, dtype=torch.bool, device=dev)
    first[[e for e in [0] + ends[:-1] if e < n]] = True
    X, R, I, Z, G, a0 = (t.double() for t in (x, r, i, z, dy, A))
    w = a0 * torch.sigmoid(R)
    a, m = torch.exp(w), torch.sqrt(-torch.expm1(2 * w))
    u, gate = torch.sigmoid(I) * X, Z * torch.sigmoid(Z)
    step = 2.0 ** -23
    c = (4 + w.abs() * (6 + 2 * R.abs())) * step
    base = (40 + 4 * (R.abs() + I.abs() + Z.abs())) * step
    h, mag = scan(a, m * u, first), scan(a, m * u.abs(), first)
    eh = scan(a, (c + base) * mag, first)
    close(y, h * gate, (eh + base * mag) * gate.abs(), "y")
    last = [e - 1 for e, k in zip(ends, lens) if k]
    at = [k for k, v in enumerate(lens) if v]
    close(state[at], h[last], eh[last], "state")
    dh, dmag = scan(a, G * gate, first, True), scan(a, (G * gate).abs(), first, True)
    ed = scan(a, (c + base) * dmag, first, True)
    before = lambda t: torch.where(first[:, None], torch.zeros_like(t), torch.cat([torch.zeros_like(t[:1]), t[:-1]]))  # noqa: E731
    si, sr, sz = torch.sigmoid(I), torch.sigmoid(R), torch.sigmoid(Z)
    close(grads["dx"], dh * m * si, (ed + base * dmag) * m * si, "dx")
    k = m * u * torch.sigmoid(-I)
    close(grads["di"], dh * k, (ed + base * dmag) * k.abs(), "di")
    pull = u * a * a / m
    e, ah = dh * (a * before(h) - pull), a * before(mag) + pull.abs()
    ee = ed * ah + dmag * (a * before(eh) + (base + c) * ah)
    kr = (a0 * sr * torch.sigmoid(-R)).abs()
    close(grads["dr"], e * a0 * sr * torch.sigmoid(-R), (ee + base * dmag * ah) * kr, "dr")
    slope = sz * (1 + Z * torch.sigmoid(-Z))
    close(grads["dz"], G * h * slope, (eh + base * mag) * (G * slope).abs() + base * mag * G.abs() * sz * (1 + Z.abs()), "dz")
    # a sum over the rows: of 8 in turn in a lane, over the waves, the tiles in 16 runs of 4
    terms = dmag * ah * sr
    close(grads["dA"], (e * sr).sum(0), ((ee + base * dmag * ah) * sr).sum(0) + (24 + n / 64 / 64) * step * terms.sum(0), "dA")
    again = mamba_hip.gated_scan_packed_bwd(dy, x, r, i, A, cu, carry, z)
    assert torch.equal(y, mamba_hip.gated_scan_packed(x, r, i, A, cu, z))
    assert all(torch.equal(grads[q], again[q]) for q in ("dx", "dr", "di", "dz", "dA"))
