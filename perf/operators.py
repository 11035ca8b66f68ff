"""Measured cases of the operators that train and serve a pre-norm Mamba-1 layer
on packed sequences: the short causal convolution and the selective scan (forward,
gradients, and single tokens on a cache addressed by slot), layer norm with its
gradients, and dropout from a counter-based generator.

``run`` computes a case in its plain form (torch operations in 32 bits, rounded
once at the end) or, with ``own`` set, through mamba_hip's entry points.  ``exact``
is the definition in 64 bits, sequences walked token by token.
"""

import functools
import math
import os
import sys

import torch

own = False
DEV = "cuda"
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _hip():
    path = os.path.join(ROOT, "burn-mamba_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mamba_hip
    return mamba_hip


# ------------------------------------------------------------------ the cases --

def listed():
    return [
        # A training step's scan at the Mamba-1 2.8B width: six documents packed
        # into one row of 8192 tokens.
        dict(name="scan_train_bf16", kind="scan_train", dtype="bf16", t=8192, s=6, pad=0, d=5120, n=16, h0=False),
        # The same in f32 at odd sizes, continuing a previous segment's states
        # (truncated backpropagation) and handing its own on.
        dict(name="scan_train_f32_odd", kind="scan_train", dtype="f32", t=1023, s=3, pad=0, d=777, n=16, h0=True),
        # Serving: nine prompts of different lengths in one call, padded to a
        # bucket, on a cache of slots.
        dict(name="scan_prompts_bf16", kind="scan_prompts", dtype="bf16", t=4000, s=9, pad=96, d=2560, n=16, slots=16),
        # One short prompt of a small model: latency.
        dict(name="scan_prompt_short_f32", kind="scan_prompts", dtype="f32", t=77, s=1, pad=0, d=512, n=16, slots=4),
        # The convolution of a training step.
        dict(name="conv_train_bf16", kind="conv_train", dtype="bf16", t=16384, s=12, pad=0, d=5120, k=4),
        # The convolution of a mixed serving batch: odd width, windows of slots.
        dict(name="conv_prompts_f32", kind="conv_prompts", dtype="f32", t=1500, s=7, pad=36, d=1000, k=3, slots=9),
        # One token for one user, and for a large batch spread over a cache.
        dict(name="token_1", kind="token", dtype="bf16", b=1, d=5120, n=16, k=4, slots=32),
        dict(name="token_256", kind="token", dtype="bf16", b=256, d=5120, n=16, k=4, slots=320),
        # Layer norm in a training step, and on the rows of a decode batch.
        dict(name="norm_train_bf16", kind="norm_train", dtype="bf16", rows=16384, cols=2560),
        dict(name="norm_rows_f32", kind="norm_fwd", dtype="f32", rows=33, cols=769),
        # Dropout with the residual sum in a training step, and alone at an odd size.
        dict(name="dropout_train_bf16", kind="dropout", dtype="bf16", rows=16384, cols=2560, p=0.1, residual=True),
        dict(name="dropout_f32_odd", kind="dropout", dtype="f32", rows=301, cols=777, p=0.25, residual=False),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["scan_train", "scan_prompts", "conv_train", "conv_prompts", "token", "norm_train", "norm_fwd",
                       "dropout"])
    dtype = rng.choice(["bf16", "f32"])
    wide = rng.choice([256, 512, 777, 1000, 1024, 2048, 2560, 5120])
    if kind == "scan_train":
        n = rng.choice([8, 16, 16, 16, 32])
        return dict(kind=kind, dtype=dtype, t=_spread(rng, 33, 8192 if n <= 16 else 2048), s=rng.randint(1, 8),
                    pad=rng.choice([0, 0, 31]), d=wide, n=n, h0=rng.random() < 0.5)
    if kind == "scan_prompts":
        s = rng.randint(1, 16)
        return dict(kind=kind, dtype=dtype, t=_spread(rng, 17, 8192), s=s, pad=rng.choice([0, 0, 57]), d=wide,
                    n=rng.choice([8, 16, 16, 16, 32, 64]) if wide <= 1024 else 16, slots=s + rng.randint(0, 8))
    if kind == "conv_train":
        return dict(kind=kind, dtype=dtype, t=_spread(rng, 64, 16384), s=rng.randint(1, 16), pad=rng.choice([0, 0, 31]),
                    d=wide, k=rng.choice([2, 3, 4, 4]))
    if kind == "conv_prompts":
        s = rng.randint(1, 16)
        return dict(kind=kind, dtype=dtype, t=_spread(rng, 17, 8192), s=s, pad=rng.choice([0, 0, 57]), d=wide,
                    k=rng.choice([2, 3, 4, 4]), slots=s + rng.randint(0, 8))
    if kind == "token":
        b = _spread(rng, 1, 256)
        return dict(kind=kind, dtype=dtype, b=b, d=wide, n=rng.choice([8, 16, 16, 16, 32, 64]), k=rng.choice([2, 3, 4, 4]),
                    slots=b + rng.randint(0, 64))
    if kind == "norm_train":
        return dict(kind=kind, dtype=dtype, rows=_spread(rng, 64, 16384), cols=_spread(rng, 100, 2560))
    if kind == "norm_fwd":
        return dict(kind=kind, dtype=dtype, rows=_spread(rng, 1, 4096), cols=_spread(rng, 100, 5120))
    return dict(kind=kind, dtype=dtype, rows=_spread(rng, 16, 16384), cols=_spread(rng, 100, 2560),
                p=rng.choice([0.05, 0.1, 0.25, 0.5]), residual=rng.random() < 0.6)


# --------------------------------------------------------------------- inputs --

class _Rand:
    """Seeded values on the GPU, in the case's type unless told otherwise."""

    def __init__(self, case, seed):
        self.io = BF16 if case["dtype"] == "bf16" else F32
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

    def dt_bias(self, d):
        """The block's initialisation: softplus^-1 of steps between 1e-3 and 0.1."""
        dt = torch.exp(self.uniform(math.log(1e-3), math.log(0.1), d))
        return dt + torch.log(-torch.expm1(-dt))


def _sequences(r, st, case):
    cuts = r.cuts(case["t"], case["s"])
    st["cu"] = torch.tensor(cuts, dtype=torch.int32, device=DEV)
    st["longest"] = max(b - a for a, b in zip(cuts, cuts[1:]))


def _scan_inputs(r, st, rows, d, n):
    """What the products around the scan leave behind: z is half of in_proj's rows,
    B and C are columns of x_proj's."""
    st["u"] = r.normal(rows, d)
    st["delta"] = r.normal(rows, d, std=0.5)
    st["z"] = r.normal(rows, 2 * d)[:, d:]
    low = -(-d // 32)
    x_dbl = r.normal(rows, low + 2 * n)
    st["B"], st["C"] = x_dbl[:, low:low + n], x_dbl[:, low + n:]
    st["A"] = -torch.exp(torch.log(torch.arange(1, n + 1, device=DEV, dtype=F32)).repeat(d, 1) + r.normal(d, n, std=0.1, dtype=F32))
    st["D"] = 1 + r.normal(d, std=0.1, dtype=F32)
    st["dt_bias"] = r.dt_bias(d)


def _leaves(st, *names):
    for k in names:
        st[k] = st[k].detach().requires_grad_()
    st["leaves"] = names


def prepare(case, seed):
    r, kind = _Rand(case, seed), case["kind"]
    st = dict(case=case)
    if kind in ("scan_train", "scan_prompts"):
        rows, d, n = case["t"] + case["pad"], case["d"], case["n"]
        _sequences(r, st, case)
        _scan_inputs(r, st, rows, d, n)
        if kind == "scan_prompts":
            st["state"] = r.normal(case["slots"], d, n, std=0.3, dtype=F32)
            st["slots"] = r.slots(case["s"], case["slots"])
            return st
        st["dy"] = r.normal(rows, d)
        names = ("u", "delta", "A", "B", "C", "D", "z", "dt_bias")
        if case["h0"]:
            st["h0"] = r.normal(case["s"], d, n, std=0.3, dtype=F32)
            st["dhT"] = r.normal(case["s"], d, n, dtype=F32)
            names += ("h0",)
        _leaves(st, *names)
    elif kind in ("conv_train", "conv_prompts"):
        rows, d, k = case["t"] + case["pad"], case["d"], case["k"]
        _sequences(r, st, case)
        st["x"] = r.normal(rows, 2 * d)[:, :d]
        st["w"] = r.uniform(-1 / math.sqrt(k), 1 / math.sqrt(k), d, k)
        st["bias"] = r.uniform(-1 / math.sqrt(k), 1 / math.sqrt(k), d)
        if kind == "conv_prompts":
            st["window"] = r.normal(case["slots"], d, k, dtype=F32)
            st["slots"] = r.slots(case["s"], case["slots"])
            return st
        st["dy"] = r.normal(rows, d)
        _leaves(st, "x", "w", "bias")
    elif kind == "token":
        b, d, n, k = (case[x] for x in ("b", "d", "n", "k"))
        _scan_inputs(r, st, b, d, n)
        st["x"] = r.normal(b, 2 * d)[:, :d]
        st["w"] = r.uniform(-1 / math.sqrt(k), 1 / math.sqrt(k), d, k)
        st["bias"] = r.uniform(-1 / math.sqrt(k), 1 / math.sqrt(k), d)
        st["window"] = r.normal(case["slots"], d, k, dtype=F32)
        st["state"] = r.normal(case["slots"], d, n, std=0.3, dtype=F32)
        st["slots"] = r.slots(b, case["slots"])
    elif kind in ("norm_train", "norm_fwd"):
        rows, cols = case["rows"], case["cols"]
        # a residual stream: channels of unlike size, rows off centre
        st["x"] = (r.normal(rows, cols, dtype=F32) * torch.exp(r.normal(cols, std=0.5, dtype=F32)) + r.normal(rows, 1, dtype=F32)).to(r.io)
        st["w"], st["b"] = 1 + r.normal(cols, std=0.1, dtype=F32), r.normal(cols, std=0.1, dtype=F32)
        if kind == "norm_train":
            st["dy"] = r.normal(rows, cols)
            _leaves(st, "x", "w", "b")
    else:
        rows, cols = case["rows"], case["cols"]
        st["x"], st["dy"] = r.normal(rows, cols), r.normal(rows, cols)
        st["rng"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), generator=r.host, dtype=torch.int64).to(DEV)
        st["p"] = case["p"]
        if case["residual"]:
            st["residual"] = r.normal(rows, cols)
            _leaves(st, "x", "residual")
        else:
            _leaves(st, "x")
    return st


# ------------------------------------------------------- through the framework --

def _own(st):
    m, kind = _hip(), st["case"]["kind"]
    if kind == "scan_train":
        y, hT = m.mamba1_scan_packed_autograd(st["u"], st["delta"], st["A"], st["B"], st["C"], st["cu"], D=st["D"], z=st["z"],
                                              delta_bias=st["dt_bias"], delta_softplus=True, initial_state=st.get("h0"),
                                              max_seqlen=st["longest"])
        outs, douts = ((y, hT), (st["dy"], st["dhT"])) if "h0" in st else ((y,), (st["dy"],))
        grads = torch.autograd.grad(outs, [st[k] for k in st["leaves"]], douts)
        return dict(zip(st["leaves"], grads), y=y, hT=hT)
    if kind == "scan_prompts":
        y = m.mamba1_scan_packed(st["u"], st["delta"], st["A"], st["B"], st["C"], st["cu"], D=st["D"], z=st["z"],
                                 delta_bias=st["dt_bias"], delta_softplus=True, state=st["state"], slots=st["slots"],
                                 max_seqlen=st["longest"])
        return dict(y=y, state=st["state"])
    if kind == "conv_train":
        y = m.conv1d_packed_autograd(st["x"], st["w"], st["cu"], st["bias"])
        return dict(zip(st["leaves"], torch.autograd.grad(y, [st[k] for k in st["leaves"]], st["dy"])), y=y)
    if kind == "conv_prompts":
        y = m.conv1d_packed(st["x"], st["w"], st["cu"], st["bias"], state=st["window"], slots=st["slots"])
        return dict(y=y, window=st["window"])
    if kind == "token":
        u = m.conv1d_step_slots(st["x"], st["window"], st["slots"], st["w"], st["bias"])
        y = m.scan_step_slots(u, st["delta"], st["A"], st["B"], st["C"], st["state"], st["slots"], D=st["D"], z=st["z"],
                              delta_bias=st["dt_bias"], delta_softplus=True)
        return dict(y=y, window=st["window"], state=st["state"])
    if kind == "norm_train":
        y = m.layer_norm_autograd(st["x"], st["w"], st["b"])
        return dict(zip(st["leaves"], torch.autograd.grad(y, [st[k] for k in st["leaves"]], st["dy"])), y=y)
    if kind == "norm_fwd":
        return m.layer_norm(st["x"], st["w"], st["b"])
    y = m.dropout_autograd(st["x"], st["p"], st["rng"], residual=st.get("residual"))
    return dict(zip(st["leaves"], torch.autograd.grad(y, [st[k] for k in st["leaves"]], st["dy"])), y=y)


# --------------------------------------------------------------- plain forms --

def _f(t):
    return t.detach().to(F32)


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20))))


def _silu(x):
    return x / (1 + torch.exp(-x))


def _dsilu(x):
    s = 1 / (1 + torch.exp(-x))
    return s * (1 + x * (1 - s))


def _rows(st, rows):
    """Of each row: its sequence (clamped), whether it is in one, its sequence's first row."""
    cu = st["cu"].long()
    t = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    live = seq < len(cu) - 1
    seq = torch.clamp(seq, max=len(cu) - 2)
    return t, seq, live, cu[seq]


def _doubling(a, b, step, longest):
    """h_t = a_t h_{t-1} + b_t by doubling: after log2 steps every row has its whole past."""
    if step >= longest:
        return b
    b2 = b.clone()
    b2[step:] += a[step:] * b[:-step]
    a2 = a.clone()
    a2[step:] *= a[:-step]
    return _doubling(a2, b2, 2 * step, longest)


def _scan_forward(st, h0):
    u, z, B, C, A, D = (_f(st[k]) for k in ("u", "z", "B", "C", "A", "D"))
    t, seq, live, start = _rows(st, u.shape[0])
    raw = _f(st["delta"]) + _f(st["dt_bias"])
    dl = _softplus(raw) * live[:, None]
    a = torch.exp(dl[:, :, None] * A)
    x = (dl * u)[:, :, None] * B[:, None, :]
    first = (live & (t == start)).nonzero()[:, 0]
    if h0 is not None:
        x[first] += a[first] * h0[seq[first]]
    af = a.clone()
    af[first] = 0
    h = _doubling(af, x, 1, st["longest"])
    pre = ((h * C[:, None, :]).sum(-1) + D * u) * live[:, None]
    cu = st["cu"].long()
    length = cu[1:] - cu[:-1]
    last = torch.clamp(cu[1:] - 1, min=0)
    empty = h0 if h0 is not None else torch.zeros_like(h[:1])
    hT = torch.where((length > 0)[:, None, None], h[last], empty)
    return dict(u=u, z=z, B=B, C=C, A=A, D=D, raw=raw, dl=dl, a=a, af=af, h=h, pre=pre, hT=hT, first=first, seq=seq, live=live,
                last=last, length=length)


def _scan_train(st):
    io = st["u"].dtype
    h0 = _f(st["h0"]) if "h0" in st else None
    f = _scan_forward(st, h0)
    dy = _f(st["dy"]) * f["live"][:, None]
    g = dy * _silu(f["z"])
    dz = dy * f["pre"] * _dsilu(f["z"])
    xr = f["C"][:, None, :] * g[:, :, None]
    if "dhT" in st:
        some = (f["length"] > 0).nonzero()[:, 0]
        xr[f["last"][some]] += _f(st["dhT"])[some]
    ar = torch.zeros_like(f["af"])
    ar[:-1] = f["af"][1:]
    dh = _doubling(ar.flip(0), xr.flip(0), 1, st["longest"]).flip(0)
    prev = torch.zeros_like(f["h"])
    prev[1:] = f["h"][:-1]
    prev[f["first"]] = 0 if h0 is None else h0[f["seq"][f["first"]]]
    da = dh * prev * f["a"]
    s = (dh * f["B"][:, None, :]).sum(-1)
    ddelta = ((da * f["A"]).sum(-1) + s * f["u"]) / (1 + torch.exp(-f["raw"]))
    out = dict(u=(s * f["dl"] + f["D"] * g).to(io), delta=ddelta.to(io), A=(da * f["dl"][:, :, None]).sum(0),
               B=(dh * (f["dl"] * f["u"])[:, :, None]).sum(1).to(io), C=(f["h"] * g[:, :, None]).sum(1).to(io),
               D=(g * f["u"]).sum(0), z=dz.to(io), dt_bias=ddelta.sum(0), y=(f["pre"] * _silu(f["z"])).to(io), hT=f["hT"])
    if h0 is not None:
        dh0 = torch.where((f["length"] > 0)[:, None, None], torch.zeros_like(h0), _f(st["dhT"]))
        dh0[f["seq"][f["first"]]] = f["a"][f["first"]] * dh[f["first"]]
        out["h0"] = dh0
    return out


def _scan_prompts(st):
    slots = st["slots"].long()
    f = _scan_forward(st, st["state"][slots])
    st["state"][slots] = f["hT"]
    return dict(y=(f["pre"] * _silu(f["z"])).to(st["u"].dtype), state=st["state"])


def _taps(st, x, k, window):
    """[rows, k, channels]: the k inputs that each row's output sees."""
    t, seq, live, start = _rows(st, x.shape[0])
    at = t[:, None] - (k - 1) + torch.arange(k, device=DEV)
    inside = at >= start[:, None]
    taps = x[torch.clamp(at, min=0)] * inside[:, :, None]
    if window is not None:
        column = torch.clamp(k + at - start[:, None], 0, k - 1)
        taps = torch.where(inside[:, :, None], taps, window[seq[:, None], :, column])
    return taps * live[:, None, None], live


def _conv_prompts(st):
    x, w, bias, k = _f(st["x"]), _f(st["w"]), _f(st["bias"]), st["w"].shape[1]
    slots, cu = st["slots"].long(), st["cu"].long()
    window = st["window"][slots]
    taps, live = _taps(st, x, k, window)
    pre = (taps * w.t()).sum(1) + bias
    at = cu[1:, None] - k + torch.arange(k, device=DEV)
    inside = at >= cu[:-1, None]
    column = torch.clamp(k + at - cu[:-1, None], 0, k - 1)
    old = window[torch.arange(len(slots), device=DEV)[:, None], :, column]
    st["window"][slots] = torch.where(inside[:, :, None], x[torch.clamp(at, min=0)], old).transpose(1, 2)
    return dict(y=(_silu(pre) * live[:, None]).to(st["x"].dtype), window=st["window"])


def _conv_train(st):
    x, w, bias, k = _f(st["x"]), _f(st["w"]), _f(st["bias"]), st["w"].shape[1]
    taps, live = _taps(st, x, k, None)
    pre = (taps * w.t()).sum(1) + bias
    g = _f(st["dy"]) * _dsilu(pre) * live[:, None]
    t, seq, live, start = _rows(st, x.shape[0])
    end = st["cu"].long()[1:][seq]
    at = t[:, None] + (k - 1) - torch.arange(k, device=DEV)
    later = g[torch.clamp(at, max=x.shape[0] - 1)] * ((at < end[:, None]) & live[:, None])[:, :, None]
    return dict(x=(later * w.t()).sum(1).to(st["x"].dtype), w=(taps * g[:, None, :]).sum(0).t().contiguous(), bias=g.sum(0),
                y=(_silu(pre) * live[:, None]).to(st["x"].dtype))


def _token(st):
    io, slots = st["x"].dtype, st["slots"].long()
    window = torch.cat([st["window"][slots][:, :, 1:], _f(st["x"])[:, :, None]], 2)
    st["window"][slots] = window
    u = _f(_silu((window * _f(st["w"])).sum(-1) + _f(st["bias"])).to(io))
    dl = _softplus(_f(st["delta"]) + _f(st["dt_bias"]))
    h = st["state"][slots] * torch.exp(dl[:, :, None] * _f(st["A"])) + (dl * u)[:, :, None] * _f(st["B"])[:, None, :]
    st["state"][slots] = h
    y = ((h * _f(st["C"])[:, None, :]).sum(-1) + _f(st["D"]) * u) * _silu(_f(st["z"]))
    return dict(y=y.to(io), window=st["window"], state=st["state"])


EPS = 1e-5


def _normed(st):
    x = _f(st["x"])
    c = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    return c * rstd, rstd, _f(st["w"]), _f(st["b"])


def _norm_fwd(st):
    xh, _, w, b = _normed(st)
    return (xh * w + b).to(st["x"].dtype)


def _norm_train(st):
    xh, rstd, w, b = _normed(st)
    dy = _f(st["dy"])
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dict(x=dx.to(st["x"].dtype), w=(dy * xh).sum(0), b=dy.sum(0), y=(xh * w + b).to(st["x"].dtype))


LOW = 0xFFFFFFFF


def _philox_round(state, _):
    """One round of Philox 4x32 (Salmon, Moraes, Dror and Shaw, 2011), words in 64-bit integers."""
    (c0, c1, c2, c3), (k0, k1) = state
    p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # modulo 2^64: the mask below drops the sign
    words = (((p1 >> 32) & LOW) ^ c1 ^ k0, p1 & LOW, ((p0 >> 32) & LOW) ^ c3 ^ k1, p0 & LOW)
    return words, ((k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW)


def _kept(shape, p, rng):
    """The elements that dropout keeps: word i % 4 of block i / 4 of the generator is at least p 2^32."""
    count = math.prod(shape)
    block = torch.arange((count + 3) // 4, device=DEV)
    same = torch.ones_like(block)
    counter = (block & LOW, (block >> 32) & LOW, same * (rng[1] & LOW), same * ((rng[1] >> 32) & LOW))
    words, _ = functools.reduce(_philox_round, range(10), (counter, (rng[0] & LOW, (rng[0] >> 32) & LOW)))
    return (torch.stack(words, 1).reshape(-1)[:count] >= math.floor(p * 2 ** 32 + 0.5)).reshape(shape)


def _dropout(st):
    io, p = st["x"].dtype, st["p"]
    kept = _kept(st["x"].shape, p, st["rng"])
    y = torch.where(kept, _f(st["x"]) * (1 / (1 - p)), 0)
    dx = torch.where(kept, _f(st["dy"]) * (1 / (1 - p)), 0).to(io)
    if "residual" in st:
        return dict(x=dx, residual=st["dy"], y=(_f(st["residual"]) + y).to(io))
    return dict(x=dx, y=y.to(io))


PLAIN = dict(scan_train=_scan_train, scan_prompts=_scan_prompts, conv_train=_conv_train, conv_prompts=_conv_prompts,
             token=_token, norm_train=_norm_train, norm_fwd=_norm_fwd, dropout=_dropout)


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["kind"]](state)


# ----------------------------------------------------------------------- work --

def work(case):
    kind, e = case["kind"], 2 if case["dtype"] == "bf16" else 4
    if kind in ("scan_train", "scan_prompts"):
        t, d, n, s = (case[k] for k in ("t", "d", "n", "s"))
        flops = t * d * (7 * n + 20)
        moved = e * t * (4 * d + 2 * n) + 4 * d * (n + 2)
        if kind == "scan_prompts":
            return dict(bytes=moved + 8 * s * d * n, flops=flops)
        # and dy read, du, ddelta, dz, dB, dC, dA, dD and the bias's gradient written
        moved += e * t * (4 * d + 2 * n) + 4 * d * (n + 2) + 4 * s * d * n * (4 if case["h0"] else 1)
        return dict(bytes=moved, flops=flops + t * d * (18 * n + 40))
    if kind in ("conv_train", "conv_prompts"):
        t, d, k = (case[x] for x in ("t", "d", "k"))
        if kind == "conv_prompts":
            return dict(bytes=2 * e * t * d + 4 * d * (k + 1) + 8 * case["s"] * d * k, flops=t * d * (2 * k + 5))
        return dict(bytes=4 * e * t * d + 8 * d * (k + 1), flops=t * d * (6 * k + 20))
    if kind == "token":
        b, d, n, k = (case[x] for x in ("b", "d", "n", "k"))
        return dict(bytes=8 * b * d * (n + k) + e * b * (4 * d + 2 * n) + 4 * d * (n + k + 3), flops=b * d * (7 * n + 2 * k + 25))
    elements, cols = case["rows"] * case["cols"], case["cols"]
    if kind == "norm_fwd":
        return dict(bytes=2 * e * elements + 8 * cols, flops=8 * elements)
    if kind == "norm_train":
        return dict(bytes=4 * e * elements + 16 * cols, flops=22 * elements)
    # the generator's 32-bit operations count as one each
    return dict(bytes=(5 if case["residual"] else 4) * e * elements, flops=60 * elements)


# ---------------------------------------------------------------- in 64 bits --

def _d(t):
    return t.detach().to(F64)


def _packed_rows(st):
    """[sequences, longest] row numbers and whether they are in the sequence."""
    cu = st["cu"].tolist()
    length = torch.tensor([b - a for a, b in zip(cu, cu[1:])], device=DEV)
    at = torch.tensor(cu[:-1], device=DEV)[:, None] + torch.arange(st["longest"], device=DEV)
    live = torch.arange(st["longest"], device=DEV) < length[:, None]
    return torch.where(live, at, torch.zeros_like(at)), live


def _exact_scan(st, h, train):
    at, live = _packed_rows(st)
    u, dy, z, B, C, A, D = (_d(st[k]) if k in st else None for k in ("u", "dy", "z", "B", "C", "A", "D"))
    raw = _d(st["delta"]) + _d(st["dt_bias"])
    dl = torch.logaddexp(raw, torch.zeros_like(raw))
    sig = torch.sigmoid(z)
    pre, before = torch.zeros_like(u), []
    for i in range(at.shape[1]):
        r, on = at[:, i], live[:, i]
        before.append(h)
        new = h * torch.exp(dl[r][:, :, None] * A) + (dl[r] * u[r])[:, :, None] * B[r][:, None, :]
        h = torch.where(on[:, None, None], new, h)
        if not train:
            before.clear()
        pre[r[on]] = ((new * C[r][:, None, :]).sum(-1) + D * u[r])[on]
    y = pre * z * sig
    if not train:
        return y, h
    g = dy * z * sig
    out = dict(y=y, hT=h, z=dy * pre * (sig + z * sig * (1 - sig)))
    inside = torch.zeros(u.shape[0], dtype=torch.bool, device=DEV)
    inside[at[live]] = True
    out["z"] = out["z"] * inside[:, None]
    du, dd, dB, dC = torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(B), torch.zeros_like(C)
    dA = torch.zeros_like(A)
    back = _d(st["dhT"]) if "dhT" in st else torch.zeros_like(h)
    for i in reversed(range(at.shape[1])):
        r, on = at[:, i], live[:, i]
        a = torch.exp(dl[r][:, :, None] * A)
        dh = back + C[r][:, None, :] * g[r][:, :, None]
        now = a * before[i] + (dl[r] * u[r])[:, :, None] * B[r][:, None, :]
        da = torch.where(on[:, None, None], dh * before[i] * a, torch.zeros_like(dh))
        s = (dh * B[r][:, None, :]).sum(-1)
        du[r[on]] = (s * dl[r] + D * g[r])[on]
        dd[r[on]] = ((da * A).sum(-1) + s * u[r])[on]
        dB[r[on]] = (dh * (dl[r] * u[r])[:, :, None]).sum(1)[on]
        dC[r[on]] = (now * g[r][:, :, None]).sum(1)[on]
        dA += (da * dl[r][:, :, None]).sum(0)
        back = torch.where(on[:, None, None], dh * a, back)
    dd = dd * torch.sigmoid(raw)
    out.update(u=du, delta=dd, B=dB, C=dC, A=dA, D=(g * u * inside[:, None]).sum(0), dt_bias=dd.sum(0))
    if "h0" in st:
        out["h0"] = back
    return out


def _exact_conv(st, window):
    """Each sequence by itself: its window, then its rows."""
    cu, x, w, bias, k = st["cu"].tolist(), _d(st["x"]), _d(st["w"]), _d(st["bias"]), st["w"].shape[1]
    y, dx, dw, db = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias)
    windows = []
    for s, (a, b) in enumerate(zip(cu, cu[1:])):
        old = torch.zeros(k, x.shape[1], dtype=F64, device=DEV) if window is None else window[s].t()
        whole = torch.cat([old, x[a:b]])
        windows.append(whole[len(whole) - k:].t())
        if a == b:
            continue
        pre = bias + sum(whole[1 + j:1 + j + b - a] * w[:, j] for j in range(k))
        sig = torch.sigmoid(pre)
        y[a:b] = pre * sig
        if "dy" in st:
            g = _d(st["dy"])[a:b] * (sig + pre * sig * (1 - sig))
            db += g.sum(0)
            dwhole = torch.zeros_like(whole)
            for j in range(k):
                dw[:, j] += (g * whole[1 + j:1 + j + b - a]).sum(0)
                dwhole[1 + j:1 + j + b - a] += g * w[:, j]
            dx[a:b] = dwhole[k:]
    return y, windows, dx, dw, db


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "scan_train":
        h = _d(st["h0"]) if "h0" in st else torch.zeros(case["s"], case["d"], case["n"], dtype=F64, device=DEV)
        return _exact_scan(st, h, True)
    if kind == "scan_prompts":
        slots, state = st["slots"].long(), _d(st["state"])
        y, h = _exact_scan(st, state[slots], False)
        state[slots] = h
        return dict(y=y, state=state)
    if kind == "conv_train":
        y, _, dx, dw, db = _exact_conv(st, None)
        return dict(x=dx, w=dw, bias=db, y=y)
    if kind == "conv_prompts":
        slots, window = st["slots"].long(), _d(st["window"])
        y, windows, _, _, _ = _exact_conv(st, window[slots])
        window[slots] = torch.stack(windows)
        return dict(y=y, window=window)
    if kind == "token":
        slots, window, state = st["slots"].long(), _d(st["window"]), _d(st["state"])
        window[slots] = torch.cat([window[slots][:, :, 1:], _d(st["x"])[:, :, None]], 2)
        pre = (window[slots] * _d(st["w"])).sum(-1) + _d(st["bias"])
        u = _d((pre * torch.sigmoid(pre)).to(st["x"].dtype))  # the scan reads the stored convolution
        raw = _d(st["delta"]) + _d(st["dt_bias"])
        dl, z = torch.logaddexp(raw, torch.zeros_like(raw)), _d(st["z"])
        h = state[slots] * torch.exp(dl[:, :, None] * _d(st["A"])) + (dl * u)[:, :, None] * _d(st["B"])[:, None, :]
        state[slots] = h
        y = ((h * _d(st["C"])[:, None, :]).sum(-1) + _d(st["D"]) * u) * z * torch.sigmoid(z)
        return dict(y=y, window=window, state=state)
    if kind in ("norm_train", "norm_fwd"):
        x, w, b = _d(st["x"]), _d(st["w"]), _d(st["b"])
        sd = torch.sqrt(x.var(1, keepdim=True, unbiased=False) + EPS)
        xh = (x - x.mean(1, keepdim=True)) / sd
        if kind == "norm_fwd":
            return xh * w + b
        dy = _d(st["dy"])
        g = dy * w
        dx = (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)) / sd
        return dict(x=dx, w=(dy * xh).sum(0), b=dy.sum(0), y=xh * w + b)
    kept = _kept_by_words(st["x"].shape, st["p"], *(int(v) % 2 ** 64 for v in st["rng"].tolist()))
    keep = kept / (1 - st["p"])
    y, dx = _d(st["x"]) * keep, _d(st["dy"]) * keep
    if "residual" in st:
        return dict(x=dx, residual=_d(st["dy"]), y=_d(st["residual"]) + y)
    return dict(x=dx, y=y)


def _kept_by_words(shape, p, seed, call):
    """The same generator in numpy's unsigned integers."""
    import numpy as np
    count = math.prod(shape)
    block = np.arange((count + 3) // 4, dtype=np.uint64)
    low, half = np.uint64(LOW), np.uint64(32)
    c = [block & low, block >> half, np.full_like(block, call & LOW), np.full_like(block, call >> 32)]
    k = [seed & LOW, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    kept = np.stack(c, 1).reshape(-1)[:count] >= np.uint64(int(p * 2 ** 32 + 0.5))
    return torch.from_numpy(kept.reshape(tuple(shape))).to(DEV).to(F64)
