"""A captured step of a Mamba-1 block after its weights have changed."""

import pytest
import torch

import mamba_hip
from test_packed_layer_gpu import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,by_slot", [(torch.float32, False), (torch.float32, True), (torch.bfloat16, True)])
def test_captured_step_follows_the_weights(dev, dtype, by_slot):
    """The replay reads the copies (the decay, the bf16 weights) where they were captured: after
    an update and a call outside the graph they hold the new values, and no other tensor."""
    layer, x, _ = make(dev)
    m, token = layer.mixer, x[:3].to(dtype)
    slots = torch.tensor([2, 0, 1], dtype=torch.int32, device=dev) if by_slot else None
    cache, eager = m.new_cache(3), m.new_cache(3)
    m.step(token, eager, slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = m.step(token, cache, slots)
    for k in range(3):
        for w in (m.a_log, m.in_proj_w, m.out_proj_w):
            w.mul_(0.8)
        for c in (cache, eager):
            c.conv_bik.fill_(0.1 * k)
            c.ssm_bir.fill_(0.3)
        want, _ = m.step(token, eager, slots)
        junk = [torch.full_like(w, 1e3, dtype=d) for w in (m.a_log, m.in_proj_w, m.out_proj_w) for d in (torch.float32, torch.bfloat16)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(cache.ssm_bir, eager.ssm_bir), k
        del junk


def test_captured_forward_follows_the_weights(dev):
    layer, x, cu = make(dev)
    m, xb, rows = layer.mixer, x.to(torch.bfloat16), x[:120].view(2, 60, -1)
    m.forward_packed(xb, cu), m.forward(rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed, (batch, _) = m.forward_packed(xb, cu), m.forward(rows)
    for k in range(3):
        for w in (m.a_log, m.in_proj_w, m.x_proj_w, m.dt_proj_w, m.out_proj_w):
            w.mul_(0.9)
        want = m.forward_packed(xb, cu), m.forward(rows)[0]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(packed, want[0]) and torch.equal(batch, want[1]), k


def test_a_weight_changes_while_its_copy_is_read(dev):
    """The new values wait for calls on other streams that still read the old ones."""
    layer, x, cu = make(dev, d_model=256)
    m, xb = layer.mixer, x.to(torch.bfloat16)
    want = m.forward_packed(xb, cu)
    torch.cuda.synchronize()
    side, big = torch.cuda.Stream(), torch.randn(4096, 4096, device=dev)
    with torch.cuda.stream(side):
        for _ in range(20):
            big = torch.tanh(big @ big)
        got = m.forward_packed(xb, cu)  # behind the products
    # the convolution and the scan parameters are the caller's own to guard: the copies are of these
    for w in (m.a_log, m.in_proj_w, m.x_proj_w, m.dt_proj_w, m.out_proj_w):
        w.mul_(0.5)
    m.forward_packed(xb, cu)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
