"""A pre-norm layer around the gated linear recurrence, every operator together: the residual's
norm, products, convolution and recurrence in training; in serving the norm's rows of 8 bits,
products with 4-bit weights and single tokens on a cache, captured and replayed."""

import pytest
import torch

import gated_oracle as go
import mamba_hip
from packed_oracle import d as f64
from packed_oracle import silu

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
D, E, K = 96, 160, 4  # model width, channels of the recurrence, taps
LENS, OUTSIDE = [70, 1, 0, 133, 5], 3
EPS = 1e-5


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def weights(g):
    """In the order of ``layer``'s leaves: norm_w, in_w [D, 4 E] (u, z, r, i), conv_w, conv_b, A, out_w."""
    return [1 + 0.2 * torch.randn(D, generator=g), torch.randn(D, 4 * E, generator=g) * D ** -0.5, torch.randn(E, K, generator=g) * 0.5,
            torch.randn(E, generator=g) * 0.1, -0.01 - 0.2 * torch.rand(E, generator=g), torch.randn(E, D, generator=g) * E ** -0.5]


def split(p):
    return p[:, :E], p[:, E:2 * E], p[:, 2 * E:3 * E], p[:, 3 * E:]


def layer(x, res, norm_w, in_w, conv_w, conv_b, A, out_w, h0, cu):
    """(out, s, final states) by the framework's operators."""
    y, s = mamba_hip.add_rms_norm_autograd(x, norm_w, res, EPS)
    u, z, r, i = split(y @ in_w.to(y.dtype))
    u = mamba_hip.conv1d_packed_autograd(u, conv_w, cu, conv_b)
    h, final = mamba_hip.gated_scan_packed_autograd(u, r, i, A, cu, z, h0)
    return h @ out_w.to(h.dtype), s, final


def plain(lens, x, res, norm_w, in_w, conv_w, conv_b, A, out_w, h0, window=None):
    """The layer in 64 bits, differentiable; rows behind the sequences are cut off from it."""
    s = res + x
    y = s / torch.sqrt((s * s).mean(1, keepdim=True) + EPS) * norm_w
    u, z, r, i = split(y @ in_w)
    a = torch.exp(A * torch.sigmoid(r))
    m = torch.sqrt(-torch.expm1(2 * A * torch.sigmoid(r)))
    rows, final, t = [], [], 0
    for q, count in enumerate(lens):
        whole = torch.cat([torch.zeros(K, E, dtype=F64) if window is None else window[q].t(), u[t:t + count]])
        v = silu(conv_b + sum(whole[1 + j:1 + j + count] * conv_w[:, j] for j in range(K)))
        h = h0[q]
        for j in range(count):
            h = a[t + j] * h + m[t + j] * torch.sigmoid(i[t + j]) * v[j]
            rows.append(h * silu(z[t + j]))
        final.append(h)
        t += count
    out = torch.stack(rows) @ out_w
    return torch.cat([out, torch.zeros(len(x) - t, D, dtype=F64)]), s, torch.stack(final)


def near(got, ref, rel, what):
    """In the 2-norm: each stage in its type's roundings (f32: sums of at most some hundred terms,
    a few hundred steps of 2^-24 in all; bf16: up to five results rounded to half a step, 2^-9,
    forward and as many backward), whose terms cancel to a tenth at most here."""
    off = float((f64(got) - ref).norm() / ref.norm())
    assert off < rel, (what, off)


def cumulative(lens, dev):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)


NAMES = ("x", "res", "norm_w", "in_w", "conv_w", "conv_b", "A", "out_w", "h0")


@pytest.mark.parametrize("io,stream,rel", [(F32, F32, 500 * 10 * 2.0 ** -24), (BF16, F32, 10 * 10 * 2.0 ** -9), (BF16, BF16, 10 * 10 * 2.0 ** -9)])
def test_training(dev, io, stream, rel):
    g, rows = gen(1), sum(LENS) + OUTSIDE
    cu = cumulative(LENS, dev)
    ins = [torch.randn(rows, D, generator=g).to(io), torch.randn(rows, D, generator=g).to(stream), *weights(g), torch.randn(len(LENS), E, generator=g)]
    outs = [torch.randn(rows, D, generator=g).to(io), torch.randn(rows, D, generator=g).to(stream), torch.randn(len(LENS), E, generator=g)]
    leaves = [t.to(dev).requires_grad_() for t in ins]
    got = layer(*leaves, cu)
    grads = torch.autograd.grad(got, leaves, [t.to(dev) for t in outs])
    again = torch.autograd.grad(layer(*leaves, cu), leaves, [t.to(dev) for t in outs])
    exact = [f64(t).requires_grad_() for t in ins]
    ref = plain(LENS, *exact)
    for a, b, what in zip(got, ref, ("out", "s", "final")):
        near(a, b.detach(), rel, what)
    assert not got[0][sum(LENS):].any()
    for a, b, c, what in zip(grads, torch.autograd.grad(ref, exact, [f64(t) for t in outs]), again, NAMES):
        near(a, b, rel, what)
        assert a.dtype == leaves[NAMES.index(what)].dtype and torch.equal(a, c), what


def test_training_step_captured(dev):
    """Forward and backward of the layer in a graph, with eager work between its replays."""
    g, rows = gen(2), sum(LENS) + OUTSIDE
    cu = cumulative(LENS, dev)
    leaves = [t.to(dev).requires_grad_() for t in (torch.randn(rows, D, generator=g).to(BF16), torch.randn(rows, D, generator=g), *weights(g),
                                                   torch.randn(len(LENS), E, generator=g))]
    dout = [torch.randn(rows, D, generator=g).to(BF16).to(dev), torch.randn(rows, D, generator=g).to(dev), torch.randn(len(LENS), E, generator=g).to(dev)]

    def step():
        return torch.autograd.grad(layer(*leaves, cu), leaves, dout)

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    for rep in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b, what in zip(grads, want, NAMES):
            assert torch.equal(a, b), (rep, what)
        step()
        torch.cuda.synchronize()


class Serving:
    """The layer with 4-bit weights on a cache of slots; q8: the norm hands on rows of 8 bits."""

    def __init__(self, dev, nslots, q8, seed=3):
        g = gen(seed)
        self.ws = [t.to(dev) for t in weights(g)]
        self.norm_w, in_w, self.conv_w, self.conv_b, self.A, out_w = self.ws
        self.q8, self.dense = q8, []
        for w, zeros in ((in_w, False), (out_w, True)):
            codes, scale, zero = mamba_hip.quantize_q4(w, 32, zeros)
            z = 8.0 if zero is None else f64(zero).repeat_interleave(32, 0)[:len(w)]
            self.dense.append((f64(codes) - z) * f64(scale).repeat_interleave(32, 0)[:len(w)])
            self.__dict__["in_w" if len(self.dense) == 1 else "out_w"] = mamba_hip.pack_linear_q4(codes, scale, zero, 32)
        self.window, self.state = torch.zeros(nslots, E, K, device=dev), torch.zeros(nslots, E, device=dev)

    def products(self, x, res):
        if self.q8:
            q, scale, s = mamba_hip.add_rms_norm_q8(x, self.norm_w, res, EPS)
            return split(mamba_hip.linear_q4(q, self.in_w, x_scale=scale, dtype=x.dtype)), s
        y, s = mamba_hip.add_rms_norm(x, self.norm_w, res, EPS)
        return split(mamba_hip.linear_q4(y, self.in_w)), s

    def prefill(self, x, res, cu, slots):
        (u, z, r, i), s = self.products(x, res)
        u = mamba_hip.conv1d_packed(u, self.conv_w, cu, self.conv_b, state=self.window, slots=slots)
        h = mamba_hip.gated_scan_packed(u, r, i, self.A, cu, z, state=self.state, slots=slots)
        return mamba_hip.linear_q4(h, self.out_w), s

    def step(self, x, res, slots):
        (u, z, r, i), s = self.products(x, res)
        u = mamba_hip.conv1d_step_slots(u, self.window, slots, self.conv_w, self.conv_b)
        h = mamba_hip.gated_step_slots(u, r, i, self.A, self.state, slots, z=z)
        return mamba_hip.linear_q4(h, self.out_w), s


def test_serving(dev):
    """Prompts of several users and then token by token are the whole sequences in 64 bits."""
    lens, more, order = [40, 7, 90], 6, [4, 0, 2]
    g, m = gen(4), Serving(dev, 6, False)
    slots = torch.tensor(order, dtype=torch.int32, device=dev)
    xs = [torch.randn(n + more, D, generator=g) for n in lens]
    rs = [torch.randn(n + more, D, generator=g) for n in lens]
    out, _ = m.prefill(torch.cat([x[:n] for x, n in zip(xs, lens)]).to(dev), torch.cat([x[:n] for x, n in zip(rs, lens)]).to(dev),
                       cumulative(lens, dev), slots)
    rows = [list(o) for o in out.split(lens)]
    for t in range(more):
        o, _ = m.step(torch.stack([x[n + t] for x, n in zip(xs, lens)]).to(dev), torch.stack([x[n + t] for x, n in zip(rs, lens)]).to(dev), slots)
        for q in range(len(lens)):
            rows[q].append(o[q])
    norm_w, _, conv_w, conv_b, A, _ = map(f64, m.ws)
    ref, _, final = plain([n + more for n in lens], f64(torch.cat(xs)), f64(torch.cat(rs)), norm_w, m.dense[0], conv_w, conv_b, A, m.dense[1],
                          torch.zeros(len(lens), E, dtype=F64))
    rel = 500 * 10 * 2.0 ** -24
    near(torch.cat([torch.stack(r) for r in rows]), ref, rel, "out")
    near(m.state[order], final, rel, "state")
    others = [k for k in range(6) if k not in order]
    assert not m.state[others].any() and not m.window[others].any()


@pytest.mark.parametrize("io,stream", [(BF16, F32), (BF16, BF16), (F32, F32)])
def test_serving_captured(dev, io, stream):
    """Tokens with rows of 8 bits from a graph, replayed with new inputs and slots, give the eager
    calls' bits; a second graph of another batch runs between."""
    g = gen(5)
    eager, graphed = Serving(dev, 9, True), Serving(dev, 9, True)
    lens = [30, 2, 65]
    first = torch.tensor([7, 1, 3], dtype=torch.int32, device=dev)
    x, res = torch.randn(sum(lens), D, generator=g).to(io).to(dev), torch.randn(sum(lens), D, generator=g).to(stream).to(dev)
    a, b = (m.prefill(x, res, cumulative(lens, dev), first) for m in (eager, graphed))
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(eager.state, graphed.state)
    graphs = []
    for n in (3, 5):
        ins = [torch.zeros(n, D, dtype=io, device=dev), torch.zeros(n, D, dtype=stream, device=dev), torch.full((n,), -1, dtype=torch.int32, device=dev)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphed.step(*ins)  # slots out of range: nothing is kept
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = graphed.step(*ins)
        graphs.append((ins, graph, outs))
    for rep in range(4):
        for ins, graph, outs in graphs:
            n = len(ins[0])
            new = [torch.randn(n, D, generator=g).to(io), torch.randn(n, D, generator=g).to(stream), torch.randperm(9, generator=g)[:n].to(torch.int32)]
            for t, v in zip(ins, new):
                t.copy_(v)
            graph.replay()
            want = eager.step(*[v.to(dev) for v in new])
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]), rep
            assert torch.equal(graphed.state, eager.state) and torch.equal(graphed.window, eager.window), rep


def test_serving_rows_of_8_bits(dev):
    """With rows of 8 bits the first product is that of the rows that they stand for."""
    g, m = gen(6), Serving(dev, 4, True)
    x, res = torch.randn(4, D, generator=g).to(dev), torch.randn(4, D, generator=g).to(dev)
    q, scale, _ = mamba_hip.add_rms_norm_q8(x, m.norm_w, res, EPS)
    (u, z, r, i), _ = m.products(x, res)
    ref = (f64(q.float()) * f64(scale)[:, None]) @ m.dense[0]
    near(torch.cat([u, z, r, i], 1), ref, 500 * 2.0 ** -24, "products")
    out, _ = m.step(x, res, None)
    # the state starts from zero: h = sqrt(1 - a^2) s(i) v
    v = silu(f64(m.conv_b) + f64(u) * f64(m.conv_w)[:, -1])
    one = go.gated([1] * 4, v, f64(r), f64(i), f64(m.A), f64(z))["y"][0] @ m.dense[1]
    near(out, one, 500 * 10 * 2.0 ** -24, "out")
