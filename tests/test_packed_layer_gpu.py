"""The Mamba-1 layer on packed sequences: every operator together, in training and in
serving, against the layer in plain 64-bit torch."""

import pytest
import torch

import mamba_hip
import packed_oracle as po

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
LENS = [37, 0, 1, 90, 64]
NAMES = ("in_proj_w", "conv_w", "conv_b", "x_proj_w", "dt_proj_w", "dt_proj_b", "a_log", "d", "out_proj_w")


def make(dev, p=0.0, d_model=48):
    g = torch.Generator()
    g.manual_seed(1)
    layer = mamba_hip.Mamba1Layer.init(mamba_hip.Mamba1Config(d_model), dev, p, g)
    layer.norm_w += 0.1 * torch.randn(d_model, generator=g).to(dev)
    layer.norm_b += 0.1 * torch.randn(d_model, generator=g).to(dev)
    x = torch.randn(sum(LENS), d_model, generator=g).to(dev)
    cu = torch.tensor([0] + torch.tensor(LENS).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    return layer, x, cu


def plain(layer, ps, x, lens, keep=None, window=None, state=None):
    """The layer in 64 bits, differentiable: (y, windows, states) of sequences that go on from
    window and state."""
    c, m = layer.mixer.cfg, dict(zip(NAMES + ("norm_w", "norm_b"), ps))
    di, r, n, k = c.d_inner, c.dt_rank, c.state_rank, c.conv_kernel
    h = torch.nn.functional.layer_norm(x, (c.d_model,), m["norm_w"], m["norm_b"], layer.eps)
    xz = h @ m["in_proj_w"]
    us, windows, t = [], [], 0
    for s, count in enumerate(lens):
        old = torch.zeros(k, di, dtype=F64) if window is None else window[s].t()
        whole = torch.cat([old, xz[t:t + count, :di]])
        windows.append(whole[len(whole) - k:].t())
        us.append(po.silu(m["conv_b"] + sum(whole[1 + j:1 + j + count] * m["conv_w"][:, j] for j in range(k))))
        t += count
    u = torch.cat(us)
    dbl = u @ m["x_proj_w"]
    dt = po.softplus(dbl[:, :r] @ m["dt_proj_w"] + m["dt_proj_b"])
    h0 = torch.zeros(len(lens), di, n, dtype=F64) if state is None else state
    pre, hT = po._core(lens, dt, dt, u, -torch.exp(m["a_log"]), dbl[:, r:r + n], dbl[:, r + n:], m["d"], h0)
    y = (pre * po.silu(xz[:, di:])) @ m["out_proj_w"]
    if keep is not None:
        y = y * keep / (1 - layer.p)
    return x + y, torch.stack(windows), hT


def params(layer):
    return [getattr(layer.mixer, k) for k in NAMES] + [layer.norm_w, layer.norm_b]


def near(got, ref, rel, what):
    """In the 2-norm: products, norms and the scan in f32, each within some hundred steps of
    2^-24 of its terms; the terms of a sum cancel to about a tenth here."""
    off = float((po.d(got) - ref).norm() / ref.norm())
    assert off < rel, (what, off)


def test_training(dev):
    layer, x, cu = make(dev, p=0.3)
    rng = torch.tensor([5, 9], device=dev)
    leaves = [t.requires_grad_() for t in params(layer)] + [x.requires_grad_()]
    y = layer.forward_packed(x, cu, max_seqlen=max(LENS), rng=rng, offset=2)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(3)).to(dev)
    grads = torch.autograd.grad(y, leaves, dy)
    keep = po.philox_kept(x.numel(), 0.3, 5, 11).reshape(x.shape).to(F64)
    ps = [po.d(t).requires_grad_() for t in leaves]
    ref, _, _ = plain(layer, ps[:-1], ps[-1], LENS, keep)
    near(y, ref.detach(), 1e-5, "y")
    for name, g, w in zip(NAMES + ("norm_w", "norm_b", "x"), grads, torch.autograd.grad(ref, ps, po.d(dy))):
        near(g, w, 5e-5, name)
    # without an rng nothing is dropped
    y = layer.forward_packed(x, cu)
    near(y, plain(layer, [po.d(t) for t in leaves[:-1]], po.d(x), LENS)[0], 1e-5, "y without dropout")


def test_training_bf16_runs(dev):
    """bf16 rows, f32 parameters: everything gets a finite gradient."""
    layer, x, cu = make(dev, p=0.1)
    leaves = [t.requires_grad_() for t in params(layer)]
    xb = x.to(BF16).requires_grad_()
    y = layer.forward_packed(xb, cu, rng=torch.tensor([1, 2], device=dev))
    assert y.dtype == BF16
    y.float().square().sum().backward()
    for t in leaves + [xb]:
        assert t.grad.dtype == t.dtype and torch.isfinite(t.grad).all() and t.grad.any()


def test_serving(dev):
    """Prompts into slots, then tokens, beside other slots that keep theirs."""
    layer, x, cu = make(dev)
    cache = layer.mixer.new_cache(8)
    for t in (cache.conv_bik, cache.ssm_bir):
        t.normal_()
    slots = torch.tensor([6, 1, 3, 0, 5], dtype=torch.int32, device=dev)
    for t in (cache.conv_bik, cache.ssm_bir):
        t[slots.long()] = 0
    others = [cache.conv_bik[[2, 4, 7]].clone(), cache.ssm_bir[[2, 4, 7]].clone()]
    ps = [po.d(t) for t in params(layer)]
    y = layer.forward_packed(x, cu, cache, slots, max(LENS))
    ref, window, state = plain(layer, ps, po.d(x), LENS)
    near(y, ref, 1e-5, "prompts")
    for k in range(3):
        # two prompts go on, one of them with several tokens; then a token for each
        token = torch.randn(5, x.shape[1], generator=torch.Generator().manual_seed(k)).to(dev)
        out, _ = layer.step(token, cache, slots)
        ref, window, state = plain(layer, ps, po.d(token), [1] * 5, window=window, state=state)
        near(out, ref, 1e-5, "token")
        more = torch.randn(7, x.shape[1], generator=torch.Generator().manual_seed(9 + k)).to(dev)
        out = layer.forward_packed(more, torch.tensor([0, 6, 7], dtype=torch.int32, device=dev), cache, slots[1:3].contiguous())
        ref, w2, s2 = plain(layer, ps, po.d(more), [6, 1], window=window[1:3], state=state[1:3])
        window, state = torch.cat([window[:1], w2, window[3:]]), torch.cat([state[:1], s2, state[3:]])
        near(out, ref, 1e-5, "piece")
    near(cache.ssm_bir[slots.long()], state, 1e-5, "states")
    assert torch.equal(cache.conv_bik[[2, 4, 7]], others[0]) and torch.equal(cache.ssm_bir[[2, 4, 7]], others[1])
    # a packed batch of equal lengths is the batch
    m, b = layer.mixer, torch.randn(3, 20, x.shape[1], generator=torch.Generator().manual_seed(20)).to(dev)
    want, _ = m.forward(b)
    got = m.forward_packed(b.reshape(60, -1), torch.tensor([0, 20, 40, 60], dtype=torch.int32, device=dev))
    near(got.reshape(b.shape), po.d(want), 1e-5, "batch")


def test_trained_parameters_are_the_ones_served(dev):
    """An update in place reaches the copies that serving keeps (A, and the bf16 weights)."""
    layer, x, cu = make(dev)
    first = [layer.forward_packed(t, cu) for t in (x, x.to(BF16))]
    for t in (layer.mixer.a_log, layer.mixer.out_proj_w, layer.mixer.in_proj_w):
        t.mul_(0.7)
    ref = plain(layer, [po.d(t) for t in params(layer)], po.d(x), LENS)[0]
    near(layer.forward_packed(x, cu), ref, 1e-5, "f32")
    y = layer.forward_packed(x.to(BF16), cu)
    # bf16 products and rows: some ten half steps of 2^-8 between x and y
    near(y, ref, 10 * 2.0 ** -8, "bf16")
    assert not torch.equal(y, first[1])
    # tokens too, with slots and without
    ps, token = [po.d(t) for t in params(layer)], x[:3]
    cache = layer.mixer.new_cache(3)
    for t in (cache.conv_bik, cache.ssm_bir):
        t.normal_()
    want, _, _ = plain(layer, ps, po.d(token), [1] * 3, window=po.d(cache.conv_bik), state=po.d(cache.ssm_bir))
    for slots in (None, torch.arange(3, dtype=torch.int32, device=dev)):
        mine = mamba_hip.Mamba1Cache(cache.conv_bik.clone(), cache.ssm_bir.clone())
        near(layer.step(token, mine, slots)[0], want, 1e-5, "token")


def test_training_step_in_a_graph(dev):
    """Forward and gradients captured, no eager graph of the leaves alive; replayed on other
    rows and other dropout masks, with eager steps between."""
    layer, x, cu = make(dev, p=0.3)
    rng, dy = torch.tensor([5, 9], device=dev), torch.randn(x.shape, generator=torch.Generator().manual_seed(4)).to(dev)
    leaves = [t.requires_grad_() for t in params(layer)] + [x.requires_grad_()]

    def step():
        y = layer.forward_packed(x, cu, rng=rng)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        with torch.no_grad():
            x.mul_(0.9)
            layer.mixer.a_log.add_(0.01)
        rng += 1
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), k


def test_two_streams_share_a_weight_copy(dev):
    """The second call finds the copy that the first has ordered behind other work."""
    layer, x, cu = make(dev, d_model=256)
    xb = x.to(BF16)
    want = layer.forward_packed(xb, cu)
    for name in NAMES:
        getattr(layer.mixer, name).mul_(1.0)  # the same values, new copies
    torch.cuda.synchronize()
    s1, s2, big = torch.cuda.Stream(), torch.cuda.Stream(), torch.randn(4096, 4096, device=dev)
    with torch.cuda.stream(s1):
        for _ in range(20):
            big = torch.tanh(big @ big)
        first = layer.forward_packed(xb, cu)
    with torch.cuda.stream(s2):
        second = layer.forward_packed(xb, cu)
    torch.cuda.synchronize()
    assert torch.equal(first, want) and torch.equal(second, want)


def test_refusals(dev):
    layer, x, cu = make(dev)
    cache = layer.mixer.new_cache(2)
    with pytest.raises(mamba_hip.MambaHipError, match="row per sequence"):
        layer.forward_packed(x, cu, cache)
    with pytest.raises(mamba_hip.MambaHipError, match="cache"):
        layer.mixer.step(x[:2], None, torch.zeros(2, dtype=torch.int32, device=dev))
    with pytest.raises(mamba_hip.MambaHipError, match="shape"):
        layer.mixer.forward_packed(x[:, :-1], cu)
    layer.mixer.d.requires_grad_()
    with pytest.raises(mamba_hip.MambaHipError, match="differentiable"):
        layer.forward_packed(x, cu, layer.mixer.new_cache(5))
    with pytest.raises(mamba_hip.MambaHipError, match="differentiable"):
        layer.step(x[:2], cache, torch.zeros(2, dtype=torch.int32, device=dev))
    with torch.no_grad():
        layer.step(x[:2], cache, torch.arange(2, dtype=torch.int32, device=dev))
