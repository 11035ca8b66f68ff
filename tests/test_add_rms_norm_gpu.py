"""RMS norm with the residual's addition, its gradients and its rows of 8 bits against plain
64-bit forms (gated_oracle)."""

import pytest
import torch

import gated_oracle as go
import mamba_hip
from packed_oracle import d as f64

pytestmark = pytest.mark.gpu
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
TYPES = [(F32, F32), (BF16, F32), (BF16, BF16), (F32, None), (BF16, None)]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def rows_of(g, rows, cols, dtype, dev, left=2, right=1):
    return torch.randn(rows, left + cols + right, generator=g).to(dtype).to(dev)[:, left:left + cols]


def make(dev, rows, cols, io, stream, seed=0):
    g = gen(seed)
    x = rows_of(g, rows, cols, io, dev)
    res = None if stream is None else rows_of(g, rows, cols, stream, dev, 0, 3)
    return x, (1 + 0.2 * torch.randn(cols, generator=g)).to(dev), res


# a thread adds the squares of at most cols / 256 + 40 elements in turn, and eight sums over
# lanes and waves; half of that relative error is the root's, and a few steps are around it
def roundings(cols):
    return 30 + cols / 256


SIZES = [(1, 1), (3, 7), (5, 100), (33, 256), (2, 513), (70, 769), (9, 1000), (40, 2560), (3, 5120), (5, 7001), (2, 20000), (3, 5121), (4, 8192), (9, 10241), (2, 16384), (1, 16385)]


@pytest.mark.parametrize("io,stream", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_forward(dev, rows, cols, io, stream):
    x, w, res = make(dev, rows, cols, io, stream)
    rstd = torch.empty(rows, device=dev)
    for weight in (w, None):
        y, s = mamba_hip.add_rms_norm(x, weight, res, 1e-5, rstd=rstd)
        es, erstd, ey = go.add_rms(x, weight, res, 1e-5)
        if stream is None:
            assert s is x
        else:
            assert s.dtype == stream
            go.close(s, es, es.abs(), 1, "s")
        assert y.dtype == io
        go.close(y, ey, ey.abs(), roundings(cols), "y")
        go.close(rstd, erstd[:, 0], erstd[:, 0], roundings(cols), "rstd")


@pytest.mark.parametrize("io,stream", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES + [(700, 300), (2000, 64)])
def test_backward(dev, rows, cols, io, stream):
    x, w, res = make(dev, rows, cols, io, stream, 1)
    rstd = torch.empty(rows, device=dev)
    _, s = mamba_hip.add_rms_norm(x, w, res, 1e-5, rstd=rstd)
    g = gen(2)
    dy, ds = rows_of(g, rows, cols, io, dev, 1, 0), rows_of(g, rows, cols, s.dtype, dev)
    for weight, more in ((w, ds), (None, None)):
        got = mamba_hip.add_rms_norm_bwd(dy, s, weight, rstd, more)
        ref = go.add_rms_bwd(dy, s, weight, rstd, more)
        # the mean's sum: cols / 256 + 40 in turn and eight between lanes, as above
        go.close(got["dx"], *ref["d"], roundings(cols), "dx")
        go.close(got["dresidual"], *ref["d"], roundings(cols), "dresidual")
        assert got["dx"].dtype == io and got["dresidual"].dtype == s.dtype
        go.close(got["dweight"], *ref["dweight"], 8 + rows, "dweight")
        again = mamba_hip.add_rms_norm_bwd(dy, s, weight, rstd, more)
        assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("io,stream", TYPES)
def test_autograd(dev, io, stream):
    rows, cols = 37, 320
    x, w, res = make(dev, rows, cols, io, stream, 3)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, *([res] if res is not None else []))]
    y, s = mamba_hip.add_rms_norm_autograd(*leaves)
    g = gen(4)
    dy, ds = torch.randn(rows, cols, generator=g).to(io).to(dev), torch.randn(rows, cols, generator=g).to(s.dtype).to(dev)
    s0, rstd, _ = go.add_rms(x, w, res, 1e-5)  # the sum as it is, which a bf16 stream has rounded
    rstd = rstd[:, 0]
    ref = go.add_rms_bwd(dy, s0, w, rstd, ds)
    if res is None:  # s is x: its gradient is added by autograd, which rounds both
        grads = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        ref = go.add_rms_bwd(dy, s0, w, rstd, None)
    else:
        grads = torch.autograd.grad((y, s), leaves, (dy, ds), retain_graph=True)
        go.close(grads[2], *ref["d"], 4 * roundings(cols), "dresidual")
        assert grads[2].dtype == stream
    go.close(grads[0], *ref["d"], 4 * roundings(cols), "dx")  # rstd is up to three of its factors
    go.close(grads[1], *ref["dweight"], 8 + rows + roundings(cols), "dweight")
    assert grads[0].dtype == io and grads[1].dtype == F32
    if res is not None:
        # the sum alone, the norm alone, one leaf alone
        only = torch.autograd.grad(s, leaves, ds, retain_graph=True)
        assert torch.equal(only[0], ds.to(io)) and torch.equal(only[2], ds) and not only[1].any()
        ref = go.add_rms_bwd(dy, s0, w, rstd, None)
        only = torch.autograd.grad(y, leaves[2], dy.expand(rows, cols), retain_graph=True)
        go.close(only[0], *ref["d"], 4 * roundings(cols), "dresidual of y")
        only = torch.autograd.grad(y.sum(), leaves[1])
        ref = go.add_rms_bwd(torch.ones_like(dy), s0, w, rstd, None)
        go.close(only[0], *ref["dweight"], 8 + rows + roundings(cols), "dweight of a sum")


@pytest.mark.parametrize("rows,cols", SIZES + [(700, 300)])
def test_backward_of_the_sum_as_it_is(dev, rows, cols):
    """The two rows of a bf16 stream in the place of their rounded sum."""
    x, w, res = make(dev, rows, cols, BF16, BF16, 14)
    s0, rstd0, _ = go.add_rms(x, w, res, 1e-5)
    rstd = torch.empty(rows, device=dev)
    mamba_hip.add_rms_norm(x, w, res, 1e-5, rstd=rstd)
    g = gen(15)
    dy, ds = rows_of(g, rows, cols, BF16, dev, 1, 0), rows_of(g, rows, cols, BF16, dev)
    for weight, more in ((w, ds), (None, None)):
        got = mamba_hip.add_rms_norm_bwd(dy, res, weight, rstd, more, x=x)
        ref = go.add_rms_bwd(dy, s0, weight, rstd0[:, 0], more)
        go.close(got["dx"], *ref["d"], 4 * roundings(cols), "dx")  # rstd is up to three of its factors
        assert got["dx"] is got["dresidual"]
        go.close(got["dweight"], *ref["dweight"], 8 + rows + roundings(cols), "dweight")


@pytest.mark.parametrize("io,stream", TYPES[:3])
def test_gradients_of_leaves_are_their_own(dev, io, stream):
    """x and residual have equal gradients of one type: no leaf's is another's memory, also where
    the same tensor is both, and a second pass adds to each."""
    x, w, res = make(dev, 20, 96, io, stream, 16)
    x, w, res = (t.contiguous().requires_grad_() for t in (x, w, res))
    for rep in (1, 2):
        y, s = mamba_hip.add_rms_norm_autograd(x, w, res)
        (y.float().sum() + 2 * s.float().sum()).backward()
        if rep == 1:
            first = [t.grad.clone() for t in (x, w, res)]
    assert x.grad.data_ptr() != res.grad.data_ptr()
    for t, g in zip((x, w, res), first):
        assert torch.equal(t.grad, 2 * g)
    x.grad.zero_()
    assert torch.equal(res.grad, 2 * first[2])
    if io == stream:
        both = res.detach().clone().requires_grad_()
        y, s = mamba_hip.add_rms_norm_autograd(both, w, both)
        (one,) = torch.autograd.grad((y, s), both, (torch.ones_like(y), torch.ones_like(s)))
        s0, rstd, _ = go.add_rms(both, w, both, 1e-5)
        ref, mag = go.add_rms_bwd(torch.ones_like(y), s0, w, rstd[:, 0], torch.ones_like(s))["d"]
        # twice the gradient, which each of the two has rounded to its type
        eps = torch.finfo(io).eps
        assert bool(((f64(one) - 2 * ref).abs() <= 2 * eps * ref.abs() + 8 * roundings(96) * 2.0 ** -23 * mag).all())


def test_gradient_by_differences(dev):
    rows, cols = 5, 40
    x, w, res = make(dev, rows, cols, F32, F32, 5)
    rstd = torch.empty(rows, device=dev)
    g = gen(6)
    dy, ds = torch.randn(rows, cols, generator=g), torch.randn(rows, cols, generator=g)
    _, s = mamba_hip.add_rms_norm(x, w, res, rstd=rstd)
    got = mamba_hip.add_rms_norm_bwd(dy.to(dev), s, w, rstd, ds.to(dev))
    for k, key in ((0, "dx"), (1, "dweight"), (2, "dresidual")):
        ins = [f64(t) for t in (x, w, res)]
        v = torch.randn(ins[k].shape, generator=g, dtype=torch.float64)

        def objective(step):
            moved = list(ins)
            moved[k] = moved[k] + step * v
            es, _, ey = go.add_rms(moved[0], moved[1], moved[2], 1e-5)
            return float((ey * f64(dy)).sum() + (es * f64(ds)).sum())

        quotient = (objective(1e-5) - objective(-1e-5)) / 2e-5
        along = float((f64(got[key]) * v).sum())
        assert abs(along - quotient) <= 1e-5 * float((f64(got[key]).abs() * v.abs()).sum()), (key, along, quotient)


@pytest.mark.parametrize("io,stream", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", [torch.int8, E4M3])
def test_eight_bits(dev, rows, cols, io, stream, dtype):
    x, w, res = make(dev, rows, cols, io, stream, 7)
    if rows > 2:  # rows of unlike size, and one of zeros
        x[0] *= 1e-3
        x[1] = 0
        if res is not None:
            res[0] *= 1e-3
            res[1] = 0
    top = 127 if dtype == torch.int8 else 448
    q, scale, s = mamba_hip.add_rms_norm_q8(x, w, res, dtype=dtype)
    es, _, ey = go.add_rms(x, w, res, 1e-5)
    if stream is not None:
        go.close(s, es, es.abs(), 1, "s")
    escale = ey.abs().amax(1) / top
    go.close(scale, escale, escale, roundings(cols) + 4, "scale")
    assert q.dtype == dtype and q.shape == x.shape
    if rows > 2:
        assert scale[1] == 0 and not q[1].view(torch.int8).any()
    # half a step of the grid at y, and the roundings of y and the scale
    y, sc = f64(q.float()) * f64(scale)[:, None], f64(scale)[:, None]
    half = sc / 2 if dtype == torch.int8 else torch.maximum(2 ** -4 * ey.abs(), 2 ** -10 * sc)
    off = (y - ey).abs() - half * (1 + 2 ** -20) - (2 * roundings(cols) + 10) * 2 ** -23 * ey.abs()
    assert bool((off <= 0).all()), float(off.max())
    assert bool((q.float().abs().amax(1)[f64(scale).to(dev) > 0] == top).all())  # the largest is the top


def test_eight_bits_of_odd_rows(dev):
    """A NaN or an infinity, values whose squares overflow, and the smallest ones."""
    cols = 300
    x = torch.randn(6, cols, generator=gen(8)).to(dev)
    x[0, 5] = float("nan")
    x[1, 7] = float("-inf")
    x[2] = 0
    x[3] = 1e-30
    x[4, 9] = 1e18
    for dtype in (torch.int8, E4M3):
        q, scale, _ = mamba_hip.add_rms_norm_q8(x, None, dtype=dtype, eps=0.0 if dtype == E4M3 else 1e-5)
        assert scale[0].isnan() and scale[1].isnan() and not q[:2].view(torch.int8).any()
        assert bool(torch.isfinite(scale[4:]).all()) and bool(torch.isfinite(q[4:].float()).all())
        if dtype == E4M3:
            assert scale[2].isnan() and not q[2].view(torch.int8).any()  # 0 / 0
        else:
            assert scale[2] == 0 and not q[2].any()
            want = 1e-30 * 1e-5 ** -0.5  # eps alone under the root
            assert abs(float(scale[3]) * 127 / want - 1) < 1e-5 and bool((q[3] == 127).all())
        assert bool((q[5].float().abs().max() == (127 if dtype == torch.int8 else 448)).all())


@pytest.mark.parametrize("cols", [300, 7001])
def test_in_place_and_shapes(dev, cols):
    x, w, res = make(dev, 6, cols, BF16, F32, 9)
    y, s = mamba_hip.add_rms_norm(x, w, res)
    r2, x2 = res.clone(), x.clone()
    y2, s2 = mamba_hip.add_rms_norm(x2, w, r2, out=x2, residual_out=r2)
    assert y2 is x2 and s2 is r2 and torch.equal(y, y2) and torch.equal(s, s2)
    y3, s3 = mamba_hip.add_rms_norm(x.reshape(2, 3, cols), w, res.reshape(2, 3, cols))
    assert y3.shape == (2, 3, cols) and torch.equal(y3.view(6, cols), y) and torch.equal(s3.view(6, cols), s)
    xb, _, rb = make(dev, 6, cols, BF16, BF16, 10)
    y, s = mamba_hip.add_rms_norm(xb, w, rb)
    x4 = xb.clone()
    y4, s4 = mamba_hip.add_rms_norm(x4, w, rb, residual_out=x4)
    assert s4 is x4 and torch.equal(s4, s) and torch.equal(y4, y)
    one = res[:1].expand(6, cols)  # a broadcast row
    assert torch.equal(mamba_hip.add_rms_norm(x, w, one)[0], mamba_hip.add_rms_norm(x, w, one.contiguous())[0])


def test_no_rows(dev):
    x, w = torch.empty(0, 8, device=dev), torch.ones(8, device=dev)
    y, s = mamba_hip.add_rms_norm(x, w, x.clone())
    assert y.shape == s.shape == (0, 8)
    q, scale, _ = mamba_hip.add_rms_norm_q8(x, w)
    assert q.shape == (0, 8) and scale.shape == (0,)
    got = mamba_hip.add_rms_norm_bwd(x, x, w, torch.empty(0, device=dev))
    assert not got["dweight"].any() and got["dx"].shape == (0, 8)


def test_captured(dev):
    x, w, res = make(dev, 300, 640, BF16, F32, 11)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, res)]
    dy, ds = torch.randn(300, 640, generator=gen(12)).to(BF16).to(dev), torch.randn(300, 640, generator=gen(13)).to(dev)

    def train():
        y, s = mamba_hip.add_rms_norm_autograd(*leaves)
        return torch.autograd.grad((y, s), leaves, (dy, ds))

    want = [g.clone() for g in train()]
    q, scale, s = mamba_hip.add_rms_norm_q8(x, w, res)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        grads = train()
        q2, scale2, s2 = mamba_hip.add_rms_norm_q8(x, w, res)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
        assert torch.equal(q, q2) and torch.equal(scale, scale2) and torch.equal(s, s2)
        train()
