"""Measured cases of the operators that a gated recurrent layer is trained and served
with: the gated linear recurrence over packed sequences (forward, gradients, and single
tokens on a cache addressed by slot), root-mean-square norm with the residual's addition
(forward, gradients, and rows of 8 bits with a scale each), and products of few rows
with weights of 4 bits.

``run`` computes a case in its plain form (torch operations in 32 bits, rounded
once at the end) or, with ``own`` set, through mamba_hip's entry points.  ``exact``
is the definition in 64 bits.
"""

import math
import os
import sys

import torch

own = False
DEV = "cuda"
F32, F64, BF16, E4M3 = torch.float32, torch.float64, torch.bfloat16, torch.float8_e4m3fn
TYPES = dict(f32=F32, bf16=BF16)
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS = 1e-5


def _hip():
    path = os.path.join(ROOT, "burn-mamba_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mamba_hip
    return mamba_hip


# ------------------------------------------------------------------ the cases --

def listed():
    return [
        # A training step's recurrence at the width of a 2560-wide layer: six documents
        # packed into one row of 8192 tokens.
        dict(name="gated_train_bf16", kind="gated_train", dtype="bf16", t=8192, s=6, pad=0, d=5120, z=True, h0=False),
        # The same in f32 at odd sizes, without the output gate, continuing a previous
        # segment's states (truncated backpropagation) and handing its own on.
        dict(name="gated_train_f32_odd", kind="gated_train", dtype="f32", t=1023, s=3, pad=0, d=777, z=False, h0=True),
        # Serving: nine prompts of different lengths in one call, padded to a bucket,
        # on a cache of slots.
        dict(name="gated_prompts_bf16", kind="gated_prompts", dtype="bf16", t=4000, s=9, pad=96, d=2560, z=True, slots=16),
        # One very long sequence of a small model.
        dict(name="gated_long_f32", kind="gated_prompts", dtype="f32", t=65537, s=1, pad=0, d=512, z=False, slots=1),
        # One token for one user, and for a large batch spread over a cache.
        dict(name="gated_token_1", kind="gated_token", dtype="bf16", b=1, d=5120, z=True, slots=32),
        dict(name="gated_token_256", kind="gated_token", dtype="bf16", b=256, d=5120, z=True, slots=320),
        # The norm of a training step: bf16 rows added to a stream kept in f32.
        dict(name="rms_train_bf16", kind="rms_train", dtype="bf16", stream="f32", rows=16384, cols=2560),
        # A prompt batch's norm for products in 8-bit floats.
        dict(name="rms_e4m3_prompts", kind="rms_q8", dtype="bf16", stream="bf16", rows=4000, cols=2560),
        # One user's token through a layer's first product, and a small odd batch through
        # a head over a vocabulary, with zero points.
        dict(name="q4_row_bf16", kind="q4", dtype="bf16", m=1, k=2560, n=10240, group=64, zero=False),
        dict(name="q4_head_bf16", kind="q4", dtype="bf16", m=7, k=2560, n=50001, group=128, zero=True),
        # f32 rows of an odd width, groups of 32.
        dict(name="q4_f32_odd", kind="q4", dtype="f32", m=3, k=800, n=1537, group=32, zero=True),
        # A decode batch: the norm hands rows of 8 bits to a layer's first product.
        dict(name="norm_q4_batch", kind="norm_q4", dtype="bf16", stream="f32", m=64, k=2560, n=10240, group=64, zero=False),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["gated_train", "gated_prompts", "gated_token", "rms_train", "rms_q8", "q4", "norm_q4"])
    dtype = rng.choice(["bf16", "f32"])
    wide = rng.choice([256, 512, 777, 1000, 1024, 2048, 2560, 5120])
    if kind == "gated_train":
        return dict(kind=kind, dtype=dtype, t=_spread(rng, 33, 8192 if dtype == "bf16" else 4096), s=rng.randint(1, 8),
                    pad=rng.choice([0, 0, 31]), d=wide, z=rng.random() < 0.6, h0=rng.random() < 0.5)
    if kind == "gated_prompts":
        s = rng.randint(1, 16)
        return dict(kind=kind, dtype=dtype, t=_spread(rng, 17, 8192 if wide > 512 else 65536), s=s, pad=rng.choice([0, 0, 57]),
                    d=wide, z=rng.random() < 0.6, slots=s + rng.randint(0, 8))
    if kind == "gated_token":
        b = _spread(rng, 1, 256)
        return dict(kind=kind, dtype=dtype, b=b, d=wide, z=rng.random() < 0.6, slots=b + rng.randint(0, 64))
    stream = "f32" if dtype == "f32" else rng.choice(["f32", "bf16"])
    if kind == "rms_train":
        return dict(kind=kind, dtype=dtype, stream=stream, rows=_spread(rng, 64, 8192), cols=_spread(rng, 100, 5120))
    if kind == "rms_q8":
        return dict(kind=kind, dtype=dtype, stream=stream, rows=_spread(rng, 1, 8192), cols=_spread(rng, 100, 5120))
    group = rng.choice([32, 64, 128])
    k = group * _spread(rng, 3, 5120 // group)
    n = _spread(rng, 100, 16384)
    if kind == "q4":
        return dict(kind=kind, dtype=dtype, m=_spread(rng, 1, 64 if dtype == "bf16" else 16), k=k, n=n, group=group,
                    zero=rng.random() < 0.5)
    return dict(kind=kind, dtype=dtype, stream=stream, m=_spread(rng, 1, 256), k=k, n=n, group=group, zero=rng.random() < 0.5)


# --------------------------------------------------------------------- inputs --

class _Rand:
    """Seeded values on the GPU, in the case's type unless told otherwise."""

    def __init__(self, case, seed):
        self.io = TYPES[case["dtype"]]
        self.gen = torch.Generator(device=DEV)
        self.gen.manual_seed(seed)
        self.host = torch.Generator()
        self.host.manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=None):
        return (torch.randn(shape, generator=self.gen, device=DEV) * std).to(dtype or self.io)

    def uniform(self, lo, hi, *shape):
        return torch.rand(shape, generator=self.gen, device=DEV) * (hi - lo) + lo

    def cuts(self, t, s):
        """Where s sequences of t tokens in all begin and end."""
        inner = torch.sort(torch.randint(0, t + 1, (s - 1,), generator=self.host))[0].tolist()
        return [0] + inner + [t]

    def slots(self, s, count):
        return torch.randperm(count, generator=self.host)[:s].to(device=DEV, dtype=torch.int32)


def _gated_inputs(r, st, rows, d, gate):
    """What the convolution and the gates' product leave behind: the gates are the halves of
    one product's rows.  A state keeps 0.9 to 0.999 of itself a token where its gate is open."""
    st["x"] = r.normal(rows, d)
    gates = r.normal(rows, 2 * d)
    st["r"], st["i"] = gates[:, :d], gates[:, d:]
    st["z"] = r.normal(rows, d) if gate else None
    st["A"] = torch.log(r.uniform(0.9, 0.999, d))


def _stream(r, st, case, rows, cols):
    """A block's rows and the residual stream: channels of unlike size."""
    size = torch.exp(r.normal(cols, std=0.5, dtype=F32))
    st["x"] = r.normal(rows, cols)
    st["res"] = (r.normal(rows, cols, dtype=F32) * size).to(TYPES[case["stream"]])
    st["w"] = 1 + r.normal(cols, std=0.1, dtype=F32)


def _weights(r, st, case):
    """A checkpoint's weights of 4 bits, as it holds them: codes of 0 to 15 [k, n], a scale for
    each group of rows and column, and zero points (8 where there are none)."""
    k, n, groups = case["k"], case["n"], case["k"] // case["group"]
    st["codes"] = torch.randint(0, 16, (k, n), generator=r.gen, device=DEV, dtype=torch.uint8)
    st["scale"] = (r.uniform(0.5, 1.5, groups, n) / (4.6 * math.sqrt(k))).to(BF16)
    st["zero"] = torch.randint(5, 11, (groups, n), generator=r.gen, device=DEV, dtype=torch.uint8) if case["zero"] else None
    if own:  # laid out once, where a program loads its weights
        st["packed"] = _hip().pack_linear_q4(st["codes"], st["scale"], st["zero"])


def _leaves(st, *names):
    for k in names:
        st[k] = st[k].detach().requires_grad_()
    st["leaves"] = names


def prepare(case, seed):
    r, kind = _Rand(case, seed), case["kind"]
    st = dict(case=case)
    if kind in ("gated_train", "gated_prompts"):
        rows, d = case["t"] + case["pad"], case["d"]
        cuts = r.cuts(case["t"], case["s"])
        st["cu"] = torch.tensor(cuts, dtype=torch.int32, device=DEV)
        st["longest"] = max(b - a for a, b in zip(cuts, cuts[1:]))
        _gated_inputs(r, st, rows, d, case["z"])
        if kind == "gated_prompts":
            st["state"] = r.normal(case["slots"], d, dtype=F32)
            st["slots"] = r.slots(case["s"], case["slots"])
            return st
        st["dy"] = r.normal(rows, d)
        names = ("x", "r", "i", "A") + (("z",) if case["z"] else ())
        if case["h0"]:
            st["h0"], st["dhT"] = r.normal(case["s"], d, dtype=F32), r.normal(case["s"], d, dtype=F32)
            names += ("h0",)
        _leaves(st, *names)
    elif kind == "gated_token":
        _gated_inputs(r, st, case["b"], case["d"], case["z"])
        st["state"] = r.normal(case["slots"], case["d"], dtype=F32)
        st["slots"] = r.slots(case["b"], case["slots"])
    elif kind in ("rms_train", "rms_q8"):
        _stream(r, st, case, case["rows"], case["cols"])
        if kind == "rms_train":
            st["dy"], st["ds"] = r.normal(case["rows"], case["cols"]), r.normal(case["rows"], case["cols"], dtype=TYPES[case["stream"]])
            _leaves(st, "x", "w", "res")
    else:
        if kind == "q4":
            st["x"] = r.normal(case["m"], case["k"])
        else:
            _stream(r, st, case, case["m"], case["k"])
        _weights(r, st, case)
    return st


# ------------------------------------------------------- through the framework --

def _own(st):
    m, kind = _hip(), st["case"]["kind"]
    if kind == "gated_train":
        y, hT = m.gated_scan_packed_autograd(st["x"], st["r"], st["i"], st["A"], st["cu"], z=st["z"], initial_state=st.get("h0"))
        outs, douts = ((y, hT), (st["dy"], st["dhT"])) if "h0" in st else ((y,), (st["dy"],))
        grads = torch.autograd.grad(outs, [st[k] for k in st["leaves"]], douts)
        return dict(zip(st["leaves"], grads), y=y, hT=hT)
    if kind == "gated_prompts":
        y = m.gated_scan_packed(st["x"], st["r"], st["i"], st["A"], st["cu"], z=st["z"], state=st["state"], slots=st["slots"])
        return dict(y=y, state=st["state"])
    if kind == "gated_token":
        y = m.gated_step_slots(st["x"], st["r"], st["i"], st["A"], st["state"], st["slots"], z=st["z"])
        return dict(y=y, state=st["state"])
    if kind == "rms_train":
        y, s = m.add_rms_norm_autograd(st["x"], st["w"], st["res"], EPS)
        return dict(zip(st["leaves"], torch.autograd.grad((y, s), [st[k] for k in st["leaves"]], (st["dy"], st["ds"]))), y=y, s=s)
    if kind == "rms_q8":
        q, scale, s = m.add_rms_norm_q8(st["x"], st["w"], st["res"], EPS, dtype=E4M3)
        return dict(q=q, scale=scale, s=s)
    if kind == "q4":
        return m.linear_q4(st["x"], st["packed"])
    q, scale, s = m.add_rms_norm_q8(st["x"], st["w"], st["res"], EPS)
    return dict(y=m.linear_q4(q, st["packed"], x_scale=scale, dtype=st["x"].dtype), s=s)


# --------------------------------------------------------------- plain forms --

def _f(t):
    return None if t is None else t.detach().to(F32)


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _silu(x):
    return x / (1 + torch.exp(-x))


def _dsilu(x):
    s = _sigmoid(x)
    return s * (1 + x * (1 - s))


def _rows(st, rows):
    """Of each row: its sequence (clamped), whether it is in one, whether it is its first."""
    cu = st["cu"].long()
    t = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    live = seq < len(cu) - 1
    seq = torch.clamp(seq, max=len(cu) - 2)
    return seq, live, live & (t == cu[seq])


def _doubling(a, b, step, longest):
    """h_t = a_t h_{t-1} + b_t by doubling: after log2 steps every row has its whole past."""
    if step >= longest:
        return b
    b2 = b.clone()
    b2[step:] += a[step:] * b[:-step]
    a2 = a.clone()
    a2[step:] *= a[:-step]
    return _doubling(a2, b2, 2 * step, longest)


def _gated(st, h0):
    x, r, i, z, A = (_f(st[k]) for k in ("x", "r", "i", "z", "A"))
    seq, live, first = _rows(st, x.shape[0])
    sr, si = _sigmoid(r), _sigmoid(i)
    la = A * sr
    a, m = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
    b = m * si * x * live[:, None]
    at = first.nonzero()[:, 0]
    if h0 is not None:
        b[at] += a[at] * h0[seq[at]]
    af = a * (live & ~first)[:, None]
    h = _doubling(af, b, 1, st["longest"])
    cu = st["cu"].long()
    some = cu[1:] > cu[:-1]
    last = torch.clamp(cu[1:] - 1, min=0)
    hT = torch.where(some[:, None], h[last], h0 if h0 is not None else torch.zeros_like(h[:1]))
    y = h if z is None else h * _silu(z)
    return dict(x=x, z=z, A=A, sr=sr, si=si, a=a, m=m, af=af, h=h, hT=hT, y=y * live[:, None], at=at, seq=seq, live=live,
                last=last, some=some)


def _gated_train(st):
    io = st["x"].dtype
    h0 = _f(st["h0"]) if "h0" in st else None
    f = _gated(st, h0)
    dy = _f(st["dy"]) * f["live"][:, None]
    g = dy.clone() if f["z"] is None else dy * _silu(f["z"])
    if "dhT" in st:
        g[f["last"][f["some"]]] += st["dhT"][f["some"]]
    ar = torch.zeros_like(f["af"])
    ar[:-1] = f["af"][1:]
    dh = _doubling(ar.flip(0), g.flip(0), 1, st["longest"]).flip(0)
    before = torch.zeros_like(f["h"])
    before[1:] = f["h"][:-1]
    before[f["at"]] = 0 if h0 is None else h0[f["seq"][f["at"]]]
    dm = dh * f["si"] * f["x"]
    dla = (dh * before - dm * f["a"] / f["m"]) * f["a"] * f["live"][:, None]
    out = dict(x=(dh * f["m"] * f["si"]).to(io), r=(dla * f["A"] * f["sr"] * (1 - f["sr"])).to(io),
               i=(dm * f["m"] * (1 - f["si"])).to(io), A=(dla * f["sr"]).sum(0), y=f["y"].to(io), hT=f["hT"])
    if f["z"] is not None:
        out["z"] = (dy * f["h"] * _dsilu(f["z"])).to(io)
    if h0 is not None:
        dh0 = torch.where(f["some"][:, None], torch.zeros_like(h0), st["dhT"])
        dh0[f["seq"][f["at"]]] = f["a"][f["at"]] * dh[f["at"]]
        out["h0"] = dh0
    return out


def _gated_prompts(st):
    slots = st["slots"].long()
    f = _gated(st, st["state"][slots])
    st["state"][slots] = f["hT"]
    return dict(y=f["y"].to(st["x"].dtype), state=st["state"])


def _gated_token(st):
    x, r, i, z, A = (_f(st[k]) for k in ("x", "r", "i", "z", "A"))
    slots = st["slots"].long()
    la = A * _sigmoid(r)
    h = st["state"][slots] * torch.exp(la) + torch.sqrt(-torch.expm1(2 * la)) * _sigmoid(i) * x
    st["state"][slots] = h
    return dict(y=(h if z is None else h * _silu(z)).to(st["x"].dtype), state=st["state"])


def _normed(st):
    s = _f(st["res"]) + _f(st["x"])
    rstd = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + EPS)
    return s, s * rstd, rstd, _f(st["w"])


def _rms_train(st):
    s, xh, rstd, w = _normed(st)
    dy = _f(st["dy"])
    g = dy * w
    d = _f(st["ds"]) + rstd * (g - xh * (g * xh).mean(1, keepdim=True))
    return dict(x=d.to(st["x"].dtype), res=d.to(st["res"].dtype), w=(dy * xh).sum(0), y=(xh * w).to(st["x"].dtype),
                s=s.to(st["res"].dtype))


def _rms_q8(st):
    s, xh, _, w = _normed(st)
    y = xh * w
    scale = y.abs().amax(1) / 448
    return dict(q=(y / scale[:, None]).to(E4M3), scale=scale, s=s.to(st["res"].dtype))


def _dense(st):
    """The weights that the codes stand for, in f32 [k, n]."""
    group = st["case"]["group"]
    wide = lambda t: _f(t).repeat_interleave(group, 0)  # noqa: E731
    return (_f(st["codes"]) - (8 if st["zero"] is None else wide(st["zero"]))) * wide(st["scale"])


def _q4(st):
    return (_f(st["x"]) @ _dense(st)).to(st["x"].dtype)


def _norm_q4(st):
    s, xh, _, w = _normed(st)
    y = xh * w
    scale = y.abs().amax(1, keepdim=True) / 127
    rows = torch.round(y / scale) * scale
    return dict(y=(rows @ _dense(st)).to(st["x"].dtype), s=s.to(st["res"].dtype))


PLAIN = dict(gated_train=_gated_train, gated_prompts=_gated_prompts, gated_token=_gated_token, rms_train=_rms_train,
             rms_q8=_rms_q8, q4=_q4, norm_q4=_norm_q4)


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["kind"]](state)


# ----------------------------------------------------------------------- work --

def work(case):
    kind, e = case["kind"], 2 if case["dtype"] == "bf16" else 4
    if kind in ("gated_train", "gated_prompts"):
        t, d, s, z = case["t"], case["d"], case["s"], 1 if case["z"] else 0
        moved, flops = e * t * d * (4 + z) + 4 * d, t * d * (25 + 8 * z)
        if kind == "gated_prompts":
            return dict(bytes=moved + 8 * s * d, flops=flops)
        # and dy read, the gradients of x, r, i, z and A written, and the states' ends
        return dict(bytes=moved + e * t * d * (4 + z) + 4 * d + 4 * s * d * (4 if case["h0"] else 1), flops=flops + t * d * (35 + 10 * z))
    if kind == "gated_token":
        b, d, z = case["b"], case["d"], 1 if case["z"] else 0
        return dict(bytes=8 * b * d + e * b * d * (4 + z) + 4 * d, flops=b * d * (25 + 8 * z))
    es = {"f32": 4, "bf16": 2}.get(case.get("stream"))
    if kind == "rms_train":
        return dict(bytes=case["rows"] * case["cols"] * (4 * e + 4 * es) + 8 * case["cols"], flops=20 * case["rows"] * case["cols"])
    if kind == "rms_q8":
        return dict(bytes=case["rows"] * (case["cols"] * (e + 2 * es + 1) + 4) + 4 * case["cols"], flops=10 * case["rows"] * case["cols"])
    m, k, n, groups = case["m"], case["k"], case["n"], case["k"] // case["group"]
    weights = k * n // 2 + groups * n * (3 if case["zero"] else 2)
    if kind == "q4":
        return dict(bytes=weights + e * m * (k + n), flops=2 * m * k * n)
    return dict(bytes=weights + m * k * (e + 2 * es) + 4 * k + e * m * n, flops=2 * m * k * n + 10 * m * k)


# ---------------------------------------------------------------- in 64 bits --

def _d(t):
    return None if t is None else t.detach().to(F64)


def _walk(a, b):
    """h_t = a_t h_{t-1} + b_t over the rows, which are cut into as many stretches as each has
    rows: all stretches walked together from zero, then what enters each from the one before."""
    t, d = a.shape
    n = max(1, math.isqrt(t))
    per = -(-t // n)
    fill = n * per - t
    a = torch.cat([a, a.new_zeros(fill, d)]).view(n, per, d)
    b = torch.cat([b, b.new_zeros(fill, d)]).view(n, per, d)
    h, p = torch.empty_like(b), torch.empty_like(a)
    h[:, 0], p[:, 0] = b[:, 0], a[:, 0]
    for j in range(1, per):
        h[:, j] = a[:, j] * h[:, j - 1] + b[:, j]
        p[:, j] = a[:, j] * p[:, j - 1]
    enters = a.new_zeros(d)
    for c in range(n):
        h[c] += p[c] * enters
        enters = h[c, -1]
    return h.view(n * per, d)[:t]


def _exact_gated(st, h0, train):
    cu = st["cu"].tolist()
    x, r, i, z, A = (_d(st[k]) for k in ("x", "r", "i", "z", "A"))
    rows, d = x.shape
    la = A * torch.sigmoid(r)
    a = torch.exp(la)
    weight = torch.sqrt(-torch.expm1(2 * la))
    b = weight * torch.sigmoid(i) * x
    keep = a.clone()
    inside = torch.zeros(rows, 1, dtype=F64, device=DEV)
    inside[:cu[-1]] = 1
    begins = [(s, lo, hi) for s, (lo, hi) in enumerate(zip(cu, cu[1:])) if hi > lo]
    for s, lo, hi in begins:
        b[lo] += a[lo] * h0[s]
        keep[lo] = 0
    h = _walk(keep, b)
    hT = h0.clone()
    for s, lo, hi in begins:
        hT[s] = h[hi - 1]
    gate = torch.ones_like(x) if z is None else z * torch.sigmoid(z)
    y = h * gate * inside
    if not train:
        return y, hT
    dy = _d(st["dy"]) * inside
    g = dy * gate
    dh0 = torch.zeros_like(h0) if "dhT" not in st else _d(st["dhT"])
    for s, lo, hi in begins:
        g[hi - 1] += dh0[s]
    shifted = torch.cat([keep[1:], keep.new_zeros(1, d)])
    dh = _walk(shifted.flip(0), g.flip(0)).flip(0) * inside
    before = torch.cat([h.new_zeros(1, d), h[:-1]])
    for s, lo, hi in begins:
        before[lo] = h0[s]
        dh0[s] = a[lo] * dh[lo]
    u = torch.sigmoid(i) * x
    # d sqrt(1 - a^2) / d log a = -a^2 / sqrt(1 - a^2)
    dla = dh * (before * a - u * a * a / weight)
    out = dict(y=y, hT=hT, x=dh * weight * torch.sigmoid(i), i=dh * weight * u * torch.sigmoid(-i),
               r=dla * la * torch.sigmoid(-r), A=(dla * torch.sigmoid(r)).sum(0))
    if z is not None:
        out["z"] = dy * h * (torch.sigmoid(z) + gate * torch.sigmoid(-z))
    if "h0" in st:
        out["h0"] = dh0
    return out


def _exact_norm(st):
    s = _d(st["res"]) + _d(st["x"])
    size = torch.sqrt(s.square().mean(1, keepdim=True) + EPS)
    return s, size, s / size * _d(st["w"])


def _exact_product(st, x):
    """Group by group: (codes - zero) summed against the rows, then scaled."""
    group, codes, scale = st["case"]["group"], _d(st["codes"]), _d(st["scale"])
    y = x.new_zeros(x.shape[0], codes.shape[1])
    for g in range(scale.shape[0]):
        part, zero = x[:, g * group:(g + 1) * group], 8.0 if st["zero"] is None else _d(st["zero"])[g]
        y += (part @ codes[g * group:(g + 1) * group] - part.sum(1, keepdim=True) * zero) * scale[g]
    return y


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "gated_train":
        h0 = _d(st["h0"]) if "h0" in st else torch.zeros(case["s"], case["d"], dtype=F64, device=DEV)
        return _exact_gated(st, h0, True)
    if kind == "gated_prompts":
        slots, state = st["slots"].long(), _d(st["state"])
        y, h = _exact_gated(st, state[slots], False)
        state[slots] = h
        return dict(y=y, state=state)
    if kind == "gated_token":
        slots, state = st["slots"].long(), _d(st["state"])
        keep = torch.exp(_d(st["A"]) * torch.sigmoid(_d(st["r"])))
        h = keep * state[slots] + torch.sqrt((1 - keep) * (1 + keep)) * torch.sigmoid(_d(st["i"])) * _d(st["x"])
        state[slots] = h
        z = _d(st["z"])
        return dict(y=h if z is None else h * z * torch.sigmoid(z), state=state)
    if kind == "q4":
        return _exact_product(st, _d(st["x"]))
    s, size, y = _exact_norm(st)
    if kind == "rms_q8":
        scale = y.abs().amax(1) / 448
        return dict(q=y / scale[:, None], scale=scale, s=s)
    if kind == "norm_q4":
        scale = y.abs().amax(1, keepdim=True) / 127
        return dict(y=_exact_product(st, torch.round(y / scale)) * scale, s=s)
    w, dy = _d(st["w"]), _d(st["dy"])
    xh = s / size
    d = _d(st["ds"]) + (dy * w - xh * (dy * w * xh).mean(1, keepdim=True)) / size
    return dict(x=d, res=d, w=(dy * xh).sum(0), y=y, s=s)
