"""The edges between two codes in the 8-bit rows of the RMS norm: q is y / scale as an f32
division gives it, rounded to the nearest code, ties to even.

Rows of +1 and -1 with eps 0 and a power of two of columns have rstd 1 exactly (the squares' sum and
its mean are whole), so y is +-weight to the bit, and the weights lie on and beside the edges.  No tolerance."""

import pytest
import torch

import mamba_hip

pytestmark = pytest.mark.gpu
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def edges(dtype):
    """The values midway between two neighbouring codes, in f32 (exact)."""
    if dtype == torch.int8:
        return torch.arange(127, dtype=F32) + 0.5
    codes = torch.arange(0x7f, dtype=torch.uint8).view(E4M3).to(F32)  # 0 .. 448
    return (codes[1:] + codes[:-1]) / 2


def codes_of(y, scale, dtype):
    t = y / scale  # f32 on the host: the nearest f32 to the quotient
    return torch.round(t).to(torch.int8) if dtype == torch.int8 else t.to(E4M3)


# 16, 64, 256 and 512 lanes a row, and rows that are not held in registers
@pytest.mark.parametrize("cols", [64, 512, 4096, 8192, 32768])
@pytest.mark.parametrize("io,stream", [(F32, F32), (BF16, BF16), (BF16, F32), (BF16, None)])
@pytest.mark.parametrize("dtype", [torch.int8, E4M3])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -98, 2.0 ** 100])  # the smallest rows that are not zeros, and large ones
def test_edges(dev, cols, io, stream, dtype, size):
    g, top = gen(cols), torch.tensor([127.0 if dtype == torch.int8 else 448.0])
    sign = torch.randint(0, 2, (3, cols), generator=g).to(F32) * 2 - 1
    at = edges(dtype)
    for _ in range(4):
        amax = (1 + torch.rand(1, generator=g)) * size
        scale = amax / top
        w = at[torch.randint(0, len(at), (cols,), generator=g)] * scale
        beside = torch.randint(-1, 2, (cols,), generator=g, dtype=torch.int32)  # the f32 below, itself, the one above
        w = torch.minimum((w.view(torch.int32) + beside).view(F32), amax)
        w[0] = amax
        x = sign.to(io).to(dev)
        res = None if stream is None else torch.zeros_like(x, dtype=stream)
        q, sc, _ = mamba_hip.add_rms_norm_q8(x, w.to(dev), res, eps=0.0, dtype=dtype)
        assert torch.equal(sc.cpu(), scale.expand(3))
        want = codes_of(sign * w, scale, dtype)
        got = q.cpu()
        off = got.view(torch.int8) != want.view(torch.int8)
        off &= ~((got.float() == 0) & (want.float() == 0))  # the sign of a zero
        assert not off.any(), (int(off.sum()), off.numel())
