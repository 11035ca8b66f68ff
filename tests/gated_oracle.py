"""Plain 64-bit forms (CPU torch) of the gated linear recurrence, RMS norm with the
residual's addition and products with 4-bit weights, and bounds on what 32-bit arithmetic may
differ from them by (``packed_oracle.close``: so many roundings of 2^-23 of the sum of the
absolute values of an output's terms, and half a step of its type).

The recurrence: the logistic function comes from a hardware exp2 and reciprocal, whose
argument v log2(e) is rounded, so its relative error is at most (3 + |v|) 2^-23; the decay's
exponent w = A s(r) then has (4 + |r|) 2^-23, and a = exp(w) |w| times that and two steps
more.  A term is multiplied by a and added once a row, so a row costs 4 + |w| (6 + 2 |r|)
roundings, and what is around it (the weight sqrt(1 - a^2) and its reciprocal, two gates,
silu and its slope) at most 40 + 4 (|r| + |i| + |z|)."""

import torch

from packed_oracle import F64, close, d  # noqa: F401


def sig(v):
    return torch.sigmoid(v)


def gated_roundings(lens, r, i, A, z=None):
    top = lambda t: float(t.nan_to_num(0, 0, 0).abs().max()) if t is not None and t.numel() else 0.0  # noqa: E731
    n = sum(lens)
    r, i, z = (None if t is None else d(t)[:n] for t in (r, i, z))
    w = (d(A) * sig(r)).abs() * (6 + 2 * r.abs()) if n else torch.zeros(1)
    return 40 + 4 * (top(r) + top(i) + top(z)) + max([0] + list(lens)) * (4 + top(w))


def gated(lens, x, r, i, A, z=None, h0=None, dy=None, dhT=None):
    """{output: (value, magnitude)}; rows behind the sequences are zero, whatever they hold."""
    rows, dim = x.shape
    x, r, i, A, z, h0, dy, dhT = map(d, (x, r, i, A, z, h0, dy, dhT))
    start = h0 if h0 is not None else torch.zeros(len(lens), dim, dtype=F64)
    n = sum(lens)
    la = A * sig(r[:n])
    a = torch.exp(la)
    m = torch.sqrt(-torch.expm1(2 * la))
    u = sig(i[:n]) * x[:n]
    gate = z[:n] * sig(z[:n]) if z is not None else torch.ones_like(u)
    res = []
    for f in (lambda t: t, torch.abs):
        before, h, hT, t = torch.zeros(n, dim, dtype=F64), torch.zeros(n, dim, dtype=F64), f(start).clone(), 0
        for s, length in enumerate(lens):
            for _ in range(length):
                before[t] = hT[s]
                hT[s] = h[t] = a[t] * hT[s] + m[t] * f(u[t])
                t += 1
        wide = lambda v: torch.cat([v, torch.zeros(rows - n, dim, dtype=F64)])  # noqa: E731
        o = dict(y=wide(h * f(gate)), hT=hT)
        if dy is not None:
            g = f(dy[:n]) * f(gate)
            back = torch.zeros_like(start) if dhT is None else f(dhT).clone()
            dh, ends = torch.zeros(n, dim, dtype=F64), n
            for s in reversed(range(len(lens))):
                for t in reversed(range(ends - lens[s], ends)):
                    dh[t] = g[t] + back[s]
                    back[s] = a[t] * dh[t]
                ends -= lens[s]
            pull = torch.where(m > 0, f(u) * a * a / m, torch.zeros_like(m))
            e = dh * (a * before - pull if not res else a * before + pull)
            o.update(dx=wide(dh * m * sig(i[:n])), di=wide(dh * m * f(u) * sig(-i[:n])), dr=wide(e * f(A) * sig(r[:n]) * sig(-r[:n])),
                     dA=(e * sig(r[:n])).sum(0), dh0=back)
            if z is not None:
                sz = sig(z[:n])
                o["dz"] = wide(f(dy[:n]) * h * (sz * (1 + f(z[:n]) * sig(-z[:n]))))
        res.append(o)
    return {k: (res[0][k], res[1][k]) for k in res[0]}


def add_rms(x, w, res, eps):
    """s, xh and y in 64 bits."""
    x, w, res = map(d, (x, w, res))
    s = x if res is None else res + x
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s, rstd, s * rstd * (w if w is not None else 1)


def add_rms_bwd(dy, s, w, rstd, ds):
    """{output: (value, magnitude)} from the stored s and rstd."""
    dy, s, w, rstd, ds = map(d, (dy, s, w, rstd, ds))
    xh = s * rstd[:, None]
    g = dy * (w if w is not None else 1)
    mean = (g * xh).mean(1, keepdim=True)
    mag = rstd[:, None] * (g.abs() + xh.abs() * (g * xh).abs().mean(1, keepdim=True))
    value = rstd[:, None] * (g - xh * mean)
    if ds is not None:
        value, mag = value + ds, mag + ds.abs()
    return dict(d=(value, mag), dweight=((dy * xh).sum(0), (dy * xh).abs().sum(0)))


def q4(x, codes, scale, zero, group, bias=None, x_scale=None):
    """(value, magnitude): the magnitude as the kernels sum, codes and zero points up to 16 higher."""
    x, scale, bias, x_scale = d(x), d(scale), d(bias), d(x_scale)
    c = codes.cpu().to(F64)
    k = torch.arange(c.shape[0]) // group
    z = torch.full_like(scale, 8.0) if zero is None else zero.cpu().to(F64)
    y = x @ ((c - z[k]) * scale[k])
    mag = x.abs() @ ((c + z[k] + 32) * scale[k].abs())
    if x_scale is not None:
        y, mag = y * x_scale[:, None], mag * x_scale.abs()[:, None]
    if bias is not None:
        y, mag = y + bias, mag + bias.abs()
    return y, mag
