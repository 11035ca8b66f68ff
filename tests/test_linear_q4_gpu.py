"""Products with weights of 4 bits against a plain 64-bit form (gated_oracle), where they can
go wrong: odd widths, short last groups, rows beyond a tile, strided rows, every type."""

import pytest
import torch

import gated_oracle as go
import mamba_hip
from packed_oracle import d as f64

pytestmark = pytest.mark.gpu
BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def weight(dev, k, n, group, zero, sdtype, seed=0):
    g = gen(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (k, n), generator=g, dtype=torch.uint8).to(dev)
    scale = ((0.5 + torch.rand(groups, n, generator=g)) * 0.02).to(sdtype).to(dev)
    z = torch.randint(0, 16, (groups, n), generator=g, dtype=torch.uint8).to(dev) if zero else None
    return codes, scale, z, mamba_hip.pack_linear_q4(codes, scale, z, group)


def rows_of(dev, rows, k, dtype, seed=1, left=3, right=2, mean=0.0):
    g = gen(seed)
    if dtype == I8:
        return torch.randint(-127, 128, (rows, left + k + right), generator=g, dtype=torch.int8).to(dev)[:, left:left + k]
    return (torch.randn(rows, left + k + right, generator=g) + mean).to(dtype).to(dev)[:, left:left + k]


# a group's terms are added one by one at worst, then the groups (the slices of k that waves
# take among them), then the bias and the scale of an int8 row: so many halves of 2^-23
def roundings(k, group):
    return (min(k, group) + -(-k // group) + 24) / 2


CASES = [(1, 64, 16, 64, False, BF16), (1, 2560, 1000, 64, False, BF16), (3, 800, 1537, 32, True, F32), (7, 1000, 77, 128, True, BF16),
         (16, 384, 33, 128, False, F32), (17, 5120, 128, 64, True, BF16), (64, 1280, 640, 64, False, BF16), (65, 130, 50, 32, True, F32),
         (130, 257, 31, 128, True, BF16), (5, 1, 1, 32, True, F32), (2, 33, 7, 32, False, BF16), (33, 2560, 300, 128, False, BF16),
         (300, 640, 96, 64, True, BF16), (4, 10240, 50, 64, True, BF16)]


@pytest.mark.parametrize("dtype", [BF16, F32, I8])
@pytest.mark.parametrize("rows,k,n,group,zero,sdtype", CASES)
def test_product(dev, rows, k, n, group, zero, sdtype, dtype):
    codes, scale, z, w = weight(dev, k, n, group, zero, sdtype)
    x = rows_of(dev, rows, k, dtype)
    xs = (torch.rand(rows, generator=gen(2)) + 0.1).to(dev) * 0.01 if dtype == I8 else None
    bias = torch.randn(n, generator=gen(3)).to(dev)
    for b, out_dtype in ((None, F32), (bias, BF16)):
        ref = go.q4(x, codes, scale, z, group, b, xs)
        y = mamba_hip.linear_q4(x, w, b, xs, dtype=out_dtype)
        assert y.dtype == out_dtype and y.shape == (rows, n)
        go.close(y, *ref, roundings(k, group), "y")
        assert torch.equal(y, mamba_hip.linear_q4(x, w, b, xs, dtype=out_dtype))
    # into a wider tensor's columns, which keeps the others
    wide = torch.full((rows, n + 5), 7.0, device=dev)
    mamba_hip.linear_q4(x, w, bias, xs, out=wide[:, 2:2 + n])
    go.close(wide[:, 2:2 + n], *go.q4(x, codes, scale, z, group, bias, xs), roundings(k, group), "out")
    assert bool((wide[:, :2] == 7).all()) and bool((wide[:, 2 + n:] == 7).all())


@pytest.mark.parametrize("dtype", [BF16, F32, I8])
@pytest.mark.parametrize("rows,k,n,group,zero,sdtype", [(33, 160, 27400, 32, True, F32), (200, 1280, 6500, 64, True, BF16),
                                                        (350, 2000, 3900, 128, False, BF16), (100, 2500, 12000, 64, False, BF16),
                                                        (47, 5000, 27400, 128, True, BF16)])
def test_many_rows_and_columns(dev, rows, k, n, group, zero, sdtype, dtype):
    codes, scale, z, w = weight(dev, k, n, group, zero, sdtype)
    x = rows_of(dev, rows, k, dtype)
    xs = (torch.rand(rows, generator=gen(2)) + 0.1).to(dev) * 0.01 if dtype == I8 else None
    bias = torch.randn(n, generator=gen(3)).to(dev)
    y = mamba_hip.linear_q4(x, w, bias, xs, dtype=F32)
    go.close(y, *go.q4(x, codes, scale, z, group, bias, xs), roundings(k, group), "y")
    assert torch.equal(y, mamba_hip.linear_q4(x, w, bias, xs, dtype=F32))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_off_centre(dev, dtype):
    """Rows with a mean beside which their spread is small: what the zero points take off is
    many times the result."""
    codes, scale, z, w = weight(dev, 1280, 100, 64, True, F32, 4)
    x = rows_of(dev, 9, 1280, dtype, 5, mean=30.0)
    go.close(mamba_hip.linear_q4(x, w, dtype=F32), *go.q4(x, codes, scale, z, 64), roundings(1280, 64), "y")


def test_f32_rows_in_full(dev):
    """Every bit of an f32 row counts: a row and the same row with its low bits changed differ
    by what those are worth."""
    k = 64
    codes = torch.full((k, 16), 8, dtype=torch.uint8, device=dev)
    codes[3, :] = 9
    w = mamba_hip.pack_linear_q4(codes, torch.ones(1, 16, device=dev))
    x = torch.zeros(3, k, device=dev)
    x[0, 3], x[1, 3], x[2, 3] = 1.0 + 2 ** -23, 1.0 - 2 ** -24, -(3.0 + 2 ** -22)
    # 16 + 9 and then 16 + 8 times x: sums of at most 25 x, each rounded once
    want = f64(x)[:, 3:4].expand(3, 16)
    go.close(mamba_hip.linear_q4(x, w), want, 25 * want.abs(), 2, "y")


def test_all_codes(dev):
    """Each code at each place of a block, alone."""
    for zero in (None, 0, 15):
        k, n = 128, 16
        codes = (torch.arange(k)[:, None] + 3 * torch.arange(n)[None]).remainder(16).to(torch.uint8).to(dev)
        z = None if zero is None else torch.full((2, n), zero, dtype=torch.uint8, device=dev)
        w = mamba_hip.pack_linear_q4(codes, torch.ones(2, n, device=dev), z)
        want = codes.float() - (8 if zero is None else zero)
        for dtype in (BF16, F32):  # whole numbers: exact
            assert torch.equal(mamba_hip.linear_q4(torch.eye(k, dtype=dtype, device=dev), w, dtype=F32), want)
        one = torch.ones(k, device=dev)
        assert torch.equal(mamba_hip.linear_q4(torch.eye(k, device=dev).to(I8), w, x_scale=one, dtype=F32), want)


def test_nonfinite_rows(dev):
    codes, scale, z, w = weight(dev, 256, 40, 64, False, BF16, 6)
    x = rows_of(dev, 20, 256, F32, 7)
    x[3, 5], x[8, 200] = float("nan"), float("inf")
    for dtype in (F32, BF16):
        y = mamba_hip.linear_q4(x.to(dtype), w)
        bad = y.isnan().any(1)
        assert bad.tolist() == [i in (3, 8) for i in range(20)] and bool(y[[3, 8]].isnan().all())
        assert torch.equal(y[~bad], mamba_hip.linear_q4(x.to(dtype).nan_to_num(0, 0, 0), w)[~bad])


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("sdtype", [F32, BF16])
def test_quantize(dev, zero_points, sdtype):
    """Each weight lies within half a step of what its code stands for (and, with scales in
    bf16, what their rounding adds at the ends), and a product with the codes is the product
    with those values."""
    wt = torch.randn(200, 48, generator=gen(8)).to(dev)
    wt[:, 5] = 0
    wt[64:128, 6] = 2.5
    codes, scale, zero = mamba_hip.quantize_q4(wt, 64, zero_points, sdtype)
    assert codes.dtype == torch.uint8 and int(codes.max()) <= 15 and scale.shape == (4, 48) and scale.dtype == sdtype
    at = torch.arange(200) // 64
    z = torch.full((4, 48), 8.0, dtype=torch.float64) if zero is None else f64(zero.float())
    stands = (f64(codes.float()) - z[at]) * f64(scale)[at]
    # with zero points the ends move by up to half a step as the zero point is rounded
    reach = 1.0 if zero_points else 0.5
    ends = 16 * torch.finfo(sdtype).eps
    assert bool(((stands - f64(wt)).abs() <= f64(scale)[at] * (reach + ends) + 1e-12).all())
    w = mamba_hip.pack_linear_q4(codes, scale, zero, 64)
    x = rows_of(dev, 4, 200, F32, 9)
    go.close(mamba_hip.linear_q4(x, w), *go.q4(x, codes, scale, zero, 64), roundings(200, 64), "y")


def test_captured_and_side_by_side(dev):
    codes, scale, z, w = weight(dev, 2560, 600, 64, True, BF16, 10)
    xs = [rows_of(dev, 5, 2560, BF16, 11 + k) for k in range(2)]
    want = [mamba_hip.linear_q4(x, w) for x in xs]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = mamba_hip.linear_q4(xs[0], w)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0])
        mamba_hip.linear_q4(xs[1], w)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(mamba_hip.linear_q4(xs[k], w))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(v, want[k]) for v in got[k])


def test_no_rows(dev):
    w = weight(dev, 64, 10, 64, False, F32)[3]
    assert mamba_hip.linear_q4(torch.empty(0, 64, device=dev), w).shape == (0, 10)
