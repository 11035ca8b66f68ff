"""Layer norm with its gradients, and dropout, against plain 64-bit forms."""

import pytest
import torch

import mamba_hip
import packed_oracle as po

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def rand(*shape, seed=0, std=1.0):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g) * std


def ln_oracle(x, w, b, eps, dy=None):
    """{output: (value, magnitude)}.  Roundings: the mean of n values in f32 partial sums is off
    by at most (n / 64 + 8) steps of the mean magnitude per value (a wave's lanes, then a
    tree), so everything is within some n / 32 + 40 steps of these magnitudes."""
    x, w, b, dy = map(po.d, (x, w, b, dy))
    n = x.shape[1]
    w = torch.ones(n, dtype=torch.float64) if w is None else w
    b = torch.zeros(n, dtype=torch.float64) if b is None else b
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    xh = c * rstd
    big = (x.abs() + x.abs().mean(1, keepdim=True)) * rstd + xh.abs()  # what xh is a difference of
    out = dict(y=(xh * w + b, big * w.abs() + b.abs()), mean=(mean[:, 0], x.abs().mean(1)), rstd=(rstd[:, 0], rstd[:, 0] * (1 + (big * xh.abs()).mean(1))))
    if dy is not None:
        g = dy * w
        m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
        a1, a2 = g.abs().mean(1, keepdim=True), (g.abs() * big).mean(1, keepdim=True)
        out["dx"] = (rstd * (g - m1 - xh * m2), rstd * (g.abs() + a1 + 2 * big * a2) * (1 + (big * xh.abs()).mean(1, keepdim=True)))
        out["dweight"] = ((dy * xh).sum(0), (dy.abs() * big * (1 + (big * xh.abs()).mean(1, keepdim=True))).sum(0))
        out["dbias"] = (dy.sum(0), dy.abs().sum(0))
    return out


LN = [(1, 1, F32, True), (1, 2560, BF16, True), (3, 7, F32, False), (33, 769, F32, True), (130, 100, BF16, True),
      (17, 128, F32, True), (65, 512, BF16, True), (40, 1000, BF16, True), (500, 257, F32, False), (9, 4097, F32, True),
      (6, 5120, BF16, True), (5, 20000, F32, True), (2, 33001, BF16, True), (1100, 2560, BF16, True), (70, 1536, F32, True),
      (37, 200, BF16, True), (300, 384, BF16, False), (65, 130, F32, True), (19, 255, F32, True)]


@pytest.mark.parametrize("rows,cols,dtype,affine", LN)
def test_layer_norm(dev, rows, cols, dtype, affine):
    x = (rand(rows, cols + 5, seed=1) * 3 + rand(rows, 1, seed=2)).to(dtype).to(dev)[:, 2:2 + cols]
    dy = rand(rows, cols + 1, seed=3).to(dtype).to(dev)[:, :cols]
    w = (1 + rand(cols, seed=4)).to(dev) if affine else None
    b = rand(cols, seed=5).to(dev) if affine else None
    ref = ln_oracle(x, w, b, 1e-5, dy)
    k = cols / 32 + 40
    mean, rstd = torch.empty(rows, device=dev), torch.empty(rows, device=dev)
    y = mamba_hip.layer_norm(x, w, b, stats=(mean, rstd))
    po.close(y, *ref["y"], k, "y")
    po.close(mean, *ref["mean"], k, "mean")
    po.close(rstd, *ref["rstd"], k, "rstd")
    assert torch.equal(mamba_hip.layer_norm(x, w, b), y)
    got = mamba_hip.layer_norm_bwd(dy, x, w, mean, rstd)
    po.close(got["dx"], *ref["dx"], 4 * k, "dx")
    po.close(got["dweight"], *ref["dweight"], 2 * k + rows, "dweight")
    po.close(got["dbias"], *ref["dbias"], rows, "dbias")
    again = mamba_hip.layer_norm_bwd(dy, x, w, mean, rstd)
    assert all(torch.equal(v, again[key]) for key, v in got.items())


def test_layer_norm_far_from_zero(dev):
    """Rows whose mean is far above their spread: the variance is not a difference of squares."""
    x = (rand(8, 300, seed=6) + 1000).to(dev)
    ref = ln_oracle(x, None, None, 1e-5)
    po.close(mamba_hip.layer_norm(x, None), *ref["y"], 300 / 32 + 40, "y")
    same = torch.full((3, 64), 5.0, device=dev)
    assert not mamba_hip.layer_norm(same, None).any()


def test_layer_norm_shapes_and_autograd(dev):
    x = rand(2, 3, 5, 96, seed=7).to(dev).requires_grad_()
    w, b = (1 + rand(96, seed=8)).to(dev).requires_grad_(), rand(96, seed=9).to(dev).requires_grad_()
    y = mamba_hip.layer_norm_autograd(x, w, b)
    y.sum().backward()  # an expanded gradient
    ref = ln_oracle(x.detach().reshape(-1, 96), w, b, 1e-5, torch.ones(30, 96))
    po.close(x.grad.reshape(-1, 96), *ref["dx"], 4 * 43, "dx")
    po.close(w.grad, *ref["dweight"], 2 * 43 + 30, "dw")
    po.close(b.grad, *ref["dbias"], 30, "db")
    # transposed rows are read through a copy; no rows; into a given output
    t = rand(64, 12, seed=10).to(dev).t()
    po.close(mamba_hip.layer_norm(t, None), *ln_oracle(t, None, None, 1e-5)["y"], 42, "transposed")
    none = torch.empty(0, 9, device=dev).requires_grad_()
    v = torch.ones(9, device=dev).requires_grad_()
    mamba_hip.layer_norm_autograd(none, v).sum().backward()
    assert none.grad.shape == (0, 9) and not v.grad.any()
    out = torch.zeros(30, 100, device=dev)[:, :96]
    mamba_hip.layer_norm(x.detach().reshape(30, 96), w.detach(), b.detach(), out=out)
    assert torch.equal(out, y.detach().reshape(30, 96))
    z = rand(4, 96, seed=11).to(dev)
    want = mamba_hip.layer_norm(z, None)
    assert torch.equal(mamba_hip.layer_norm(z, None, out=z), want) and torch.equal(z, want)


@pytest.mark.parametrize("shape,p,dtype,residual", [((1,), 0.5, F32, False), ((7, 33), 0.1, BF16, True), ((3, 5, 8), 0.25, F32, True),
                                                    ((301, 77), 0.9, BF16, False), ((64, 64), 0.0, F32, True), ((9, 11), 1.0, F32, True),
                                                    ((5000,), 0.3, BF16, True)])
def test_dropout(dev, shape, p, dtype, residual):
    x = rand(*shape, seed=12).to(dtype).to(dev)
    r = rand(*shape, seed=13).to(dtype).to(dev) if residual else None
    seed, call, offset = -0x123456789abcdef, 2 ** 63 - 2, 5  # the call number wraps
    rng = torch.tensor([seed, call], device=dev)
    kept = po.philox_kept(x.numel(), p, seed % 2 ** 64, (call + offset) % 2 ** 64).reshape(shape)
    ref = torch.where(kept, po.d(x) / (1 - p) if p < 1 else po.d(x), torch.zeros((), dtype=torch.float64))
    mag = ref.abs() + (po.d(r).abs() if residual else 0)
    ref = ref + (po.d(r) if residual else 0)
    y = mamba_hip.dropout(x, p, rng, offset, r)
    po.close(y, ref, mag, 2, "y")
    if not residual:
        assert torch.equal(y.cpu() != 0, kept & (x.cpu() != 0))
    # rows of wider tensors give the same elements the same mask
    if len(shape) == 2:
        wide = torch.zeros(shape[0], shape[1] + 3, dtype=dtype, device=dev)
        wide[:, 1:-2] = x
        assert torch.equal(mamba_hip.dropout(wide[:, 1:-2], p, rng, offset, r), y)
        mamba_hip.dropout(x, p, rng, offset, r, out=wide[:, 1:-2])
        assert torch.equal(wide[:, 1:-2], y) and not wide[:, 0].any() and not wide[:, -2:].any()
    assert torch.equal(mamba_hip.dropout(x, p, rng, offset, r, out=x), y)  # in place


def test_dropout_gradient_and_masks(dev):
    x, r = rand(40, 50, seed=14).to(dev).requires_grad_(), rand(40, 50, seed=15).to(dev).requires_grad_()
    rng = torch.tensor([3, 4], device=dev)
    y = mamba_hip.dropout_autograd(x, 0.4, rng, 1, r)
    dy = rand(40, 50, seed=16).to(dev)
    gx, gr = torch.autograd.grad(y, [x, r], dy)
    kept = (y - r).detach() != 0
    assert torch.equal(gx != 0, kept) and torch.equal(gr, dy)
    po.close(gx, po.d(dy) * kept.cpu() / 0.6, po.d(dy).abs(), 2, "dx")
    # other calls, other masks; the share that is kept is 1 - p within six deviations
    many = torch.ones(1 << 20, device=dev)
    a, b = mamba_hip.dropout(many, 0.4, rng, 0), mamba_hip.dropout(many, 0.4, rng, 1)
    assert not torch.equal(a, b)
    for m in (a, b):
        assert abs(float((m != 0).float().mean()) - 0.6) < 6 * (0.24 / 2 ** 20) ** 0.5
    assert abs(float(((a != 0) & (b != 0)).float().mean()) - 0.36) < 6 * (0.36 * 0.64 / 2 ** 20) ** 0.5
    # dropped infinities are dropped
    many[:] = float("inf")
    d = mamba_hip.dropout(many, 0.4, rng, 0)
    assert torch.equal(d == 0, a == 0) and not d.isnan().any()
    # a state that moves on before the backward has run is refused by autograd
    y = mamba_hip.dropout_autograd(x, 0.4, rng, 1)
    rng[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    assert mamba_hip.dropout(torch.empty(0, 3, device=dev), 0.5, rng).shape == (0, 3)


def test_in_place(dev):
    x, r = (torch.randn(37, 90, generator=torch.Generator().manual_seed(i)).to(dev) for i in (31, 32))
    w = torch.linspace(-1, 1, 90, device=dev)
    y = x.clone()
    assert torch.equal(mamba_hip.layer_norm(y, w, out=y), mamba_hip.layer_norm(x, w))
    rng = torch.tensor([5, 6], device=dev)
    want = mamba_hip.dropout(x, 0.3, rng, residual=r)
    for k in range(2):
        mine = [x.clone(), r.clone()]
        assert torch.equal(mamba_hip.dropout(mine[0], 0.3, rng, residual=mine[1], out=mine[k]), want)


def test_graph(dev):
    """A captured step draws a new mask at each replay after the state moved on."""
    x, r, dy = (rand(300, 96, seed=s).to(BF16).to(dev) for s in (17, 18, 19))
    w, b = (1 + rand(96, seed=20)).to(dev), rand(96, seed=21).to(dev)
    rng = torch.tensor([11, 0], device=dev)
    mean, rstd = torch.empty(300, device=dev), torch.empty(300, device=dev)

    def work():
        y = mamba_hip.layer_norm(x, w, b, stats=(mean, rstd))
        o = mamba_hip.dropout(y, 0.2, rng, 7, r)
        g = mamba_hip.layer_norm_bwd(mamba_hip.dropout(dy, 0.2, rng, 7), x, w, mean, rstd)
        return [o, g["dx"], g["dweight"], g["dbias"]]

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    seen = []
    for k in range(3):
        x.copy_(rand(300, 96, seed=30 + k))
        rng[1] += 1
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in captured]
        want = work()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, want)), k
        seen.append(got[0])
    assert not torch.equal(seen[0], seen[1])
