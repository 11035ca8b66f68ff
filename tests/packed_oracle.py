"""Plain 64-bit forms (CPU torch) of the packed convolution, scan and layer norm, and
bounds on what 32-bit arithmetic may differ from them by.

The scan's bound: run on the inputs' absolute values the same formulas give, for each
output, the sum M of the absolute values of its terms.  A term passes through at most
4 roundings per row of its sequence (the decay's argument and exp, two in the update)
and some 40 around it (softplus, the gate, the sums over states and channels), each at
most 2^-23 (the hardware exp, log and reciprocal are within one step), so an output is
within (40 + 4 L) 2^-23 M before it is stored, L the longest sequence, and half a step
of its type after."""

import torch

F64 = torch.float64


def d(t):
    return None if t is None else t.detach().cpu().to(F64)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, ref, mag, roundings, what):
    """|got - ref| <= half a step of got's type |ref| + roundings 2^-23 mag, elementwise."""
    g = d(got)
    tol = half_step(got.dtype) * ref.abs() * (1 + 2 ** -8) + roundings * 2.0 ** -23 * mag + 1e-37
    bad = ~((g - ref).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float(((g - ref).abs() / tol).nan_to_num(1e9).max()):.3g} times the bound")


def silu(x):
    return x * torch.sigmoid(x)


def dsilu(x):
    s = torch.sigmoid(x)
    return s * (1 + x * (1 - s))


def softplus(x):
    return torch.logaddexp(x, torch.zeros_like(x))


def _core(lens, d1, d2, u, A, B, C, D, h0):
    """pre [rows, d] and the final states; d1 decays, d2 scales the input."""
    pre, last, t = [], [], 0
    for s, n in enumerate(lens):
        h = h0[s]
        for _ in range(n):
            h = h * torch.exp(d1[t][:, None] * A) + (d2[t] * u[t])[:, None] * B[t][None]
            pre.append((h * C[t][None]).sum(-1) + D * u[t])
            t += 1
        last.append(h)
    pre += [torch.zeros_like(u[0])] * (u.shape[0] - t)
    return torch.stack(pre) if pre else torch.zeros_like(u), torch.stack(last) if last else h0


def scan(lens, u, delta, A, B, C, D=None, z=None, bias=None, sp=False, h0=None, dy=None, dhT=None):
    """{output: (value, magnitude)} of the packed scan, and of its gradients where dy is given.
    Rows behind the sequences are zero."""
    rows, n = u.shape[0], A.shape[1]
    total = sum(lens)
    live = torch.zeros(rows, 1, dtype=F64)
    live[:total] = 1
    u, delta, A, B, C, D, z, bias, h0, dy, dhT = map(d, (u, delta, A, B, C, D, z, bias, h0, dy, dhT))
    # what rows of no sequence hold does not matter: it may be anything
    wipe = lambda t: None if t is None else torch.where(live > 0, t, torch.zeros_like(t))  # noqa: E731
    u, delta, B, C, z, dy = map(wipe, (u, delta, B, C, z, dy))
    raw = delta + (bias if bias is not None else 0)
    dt = softplus(raw) if sp else raw
    D0 = D if D is not None else torch.zeros(u.shape[1], dtype=F64)
    h0_ = h0 if h0 is not None else torch.zeros(len(lens), u.shape[1], n, dtype=F64)
    gate = silu(z) if z is not None else torch.ones_like(u)
    out = {}
    res = []
    for absolute in (False, True):
        f = (lambda t: t.abs()) if absolute else (lambda t: t)
        d2 = f(dt).clone()
        ins = [dt.clone(), d2, f(u).clone(), A.clone(), f(B).clone(), f(C).clone(), f(D0).clone(), f(h0_).clone()]
        for t in ins:
            t.requires_grad_(dy is not None)
        pre, hT = _core(lens, *ins)
        r = dict(y=(pre * f(gate)).detach(), hT=hT.detach())
        if dy is not None:
            e = f(dy) * f(gate)
            obj = (pre * e).sum() + ((hT * f(dhT)).sum() if dhT is not None else 0)
            g1, g2, gu, gA, gB, gC, gD, gh = torch.autograd.grad(obj, ins, allow_unused=True)
            zero = lambda g, t: torch.zeros_like(t) if g is None else g  # noqa: E731
            g1, g2, gu, gA, gB, gC, gD, gh = (zero(g, t) for g, t in zip((g1, g2, gu, gA, gB, gC, gD, gh), ins))
            dd = f(g1) + g2
            if sp:
                dd = dd * torch.sigmoid(raw)
            dd = dd * live
            r.update(du=gu, ddelta=dd, dA=f(gA), dB=gB, dC=gC, dD=gD, dbias=dd.sum(0), dh0=gh)
            if z is not None:
                # silu' = s (1 + z (1 - s)) is a difference where z < 0 and vanishes at z = -1.28,
                # so its terms, s and s |z| (1 - s), are what the roundings are relative to
                sg = torch.sigmoid(z)
                slope = sg * (1 + z.abs() * (1 - sg)) if absolute else dsilu(z)
                r["dz"] = f(dy) * pre.detach() * slope * live
        res.append(r)
    for k in res[0]:
        out[k] = (res[0][k], res[1][k])
    return out


def conv(lens, x, w, bias=None, act=True, window=None, dout=None):
    """{output: (value, magnitude)} of the packed convolution; window [sequences, c, K]."""
    rows, (c, k) = x.shape[0], w.shape
    x, w, bias, window, dout = map(d, (x, w, bias, window, dout))
    b = bias if bias is not None else torch.zeros(c, dtype=F64)
    res = []
    for absolute in (False, True):
        f = (lambda t: t.abs()) if absolute else (lambda t: t)
        y, wins = torch.zeros(rows, c, dtype=F64), []
        dx, dw, db = torch.zeros(rows, c, dtype=F64), torch.zeros(c, k, dtype=F64), torch.zeros(c, dtype=F64)
        t = 0
        for s, n in enumerate(lens):
            old = window[s].t() if window is not None else torch.zeros(k, c, dtype=F64)
            real = torch.cat([old, x[t:t + n]])
            whole = f(real)
            wins.append(real[len(real) - k:].t())
            if n:
                pre = b + sum(real[1 + j:1 + j + n] * w[:, j] for j in range(k))
                mag = f(b) + sum(whole[1 + j:1 + j + n] * f(w)[:, j] for j in range(k))
                # |silu'| <= 1.1: what the roundings of pre move the output by
                y[t:t + n] = (silu(pre) if act else pre) if not absolute else 1.1 * mag
                if dout is not None:
                    g = dout[t:t + n] * (dsilu(pre) if act else 1)
                    if absolute:  # |silu''| <= 0.5
                        g = dout[t:t + n].abs() * (1.1 + 0.5 * mag)
                    db += g.sum(0)
                    dwhole = torch.zeros_like(whole)
                    for j in range(k):
                        dw[:, j] += (g * whole[1 + j:1 + j + n]).sum(0)
                        dwhole[1 + j:1 + j + n] += g * f(w)[:, j]
                    dx[t:t + n] = dwhole[k:]
            t += n
        res.append(dict(y=y, window=torch.stack(wins) if wins else torch.zeros(0, c, k, dtype=F64), dx=dx, dw=dw, dbias=db))
    return {key: (res[0][key], res[1][key]) for key in res[0]}


def philox_kept(count, p, seed, call):
    """Which of `count` elements dropout keeps, in Python integers."""
    out, low = [], 0xFFFFFFFF
    for block in range((count + 3) // 4):
        c = [block & low, block >> 32, call & low, (call >> 32) & low]
        k = [seed & low, (seed >> 32) & low]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1], a & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        out += [w >= int(p * 2 ** 32 + 0.5) for w in c]
    return torch.tensor(out[:count])
