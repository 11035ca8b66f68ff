"""The copies that serving keeps beside a weight (its decay, its type, its layout): where
they lie and when they are made again.  On the CPU: no kernel is reached."""

import copy
import io

import pytest
import torch

import mamba_hip
from mamba_hip import mamba1, step


def block(seed=0):
    g = torch.Generator()
    g.manual_seed(seed)
    return mamba_hip.Mamba1Config(16).init("cpu", g)


COPIES = [(lambda m: mamba1._decay(m.a_log), lambda m: m.a_log, lambda w: -torch.exp(w)),
          (lambda m: mamba1._cast(m.out_proj_w, torch.bfloat16), lambda m: m.out_proj_w, lambda w: w.to(torch.bfloat16)),
          (lambda m: mamba1._wt(m.in_proj_w, "_mamba_t_res", 32), lambda m: m.in_proj_w, lambda w: w[:, 32:].t())]


@pytest.mark.parametrize("copy,weight,formula", COPIES)
def test_a_copy_is_made_again_where_it_is(copy, weight, formula):
    """A captured graph holds the copy's address: after an update of the weight the copy has
    the new values at the old place, and its memory was not given back."""
    m = block()
    first = copy(m)
    at = first.data_ptr()
    for _ in range(2):
        weight(m).mul_(0.5)
        again = copy(m)
        assert again.data_ptr() == at and torch.equal(again, formula(weight(m)))
        assert torch.equal(first, again)
    with torch.inference_mode():
        weight(m).mul_(0.5)
        assert copy(m).data_ptr() == at and torch.equal(first, formula(weight(m)))


def test_inference_mode_copies():
    """Weights made under inference mode are made again in place too, in the mode and out of
    it, after drop_derived."""
    with torch.inference_mode():
        m = block()
        first = mamba1._decay(m.a_log)
        at = first.data_ptr()
        m.a_log.mul_(0.5)
        step.drop_derived(m.a_log)
        assert mamba1._decay(m.a_log).data_ptr() == at and torch.equal(first, -torch.exp(m.a_log))
        m.a_log.mul_(0.5)
    step.drop_derived(m.a_log)
    assert mamba1._decay(m.a_log).data_ptr() == at and torch.equal(first, -torch.exp(m.a_log))


def test_copies_that_stay_apart():
    """One that autograd follows and one that is the weight's own memory are not written
    over: the weight's new storage leaves the old one, which may have another owner."""
    w = torch.randn(8, 4).t().requires_grad_()
    make = lambda t: (2 * t).contiguous()  # noqa: E731
    first = step._derived(w, "_mamba_test", make)
    value = first.detach().clone()
    with torch.no_grad():
        w.mul_(3)
    assert step._derived(w, "_mamba_test", make).data_ptr() != first.data_ptr() and torch.equal(first, value)
    owner = torch.randn(4, 8)
    w, kept = owner.t(), owner.clone()
    view = step._derived(w, "_mamba_test", lambda t: t.t().contiguous())
    assert view.data_ptr() == owner.data_ptr()
    w.data = torch.randn(4, 8).t()
    w.mul_(1)
    got = step._derived(w, "_mamba_test", lambda t: t.t().contiguous())
    assert torch.equal(got, w.t()) and torch.equal(owner, kept)


def test_a_copied_block_has_its_own_copies():
    """copy.deepcopy takes a tensor's attributes along and begins its version counter again:
    the decay of a block copied from a copied one, after an update that nothing served since."""
    m = copy.deepcopy(block())
    assert m.a_log._version == copy.deepcopy(m.a_log)._version  # what the counter alone cannot tell apart
    mamba1._decay(m.a_log)
    m.a_log.mul_(0.5)
    other = copy.deepcopy(m)
    assert torch.equal(other.A, -torch.exp(m.a_log))
    m.a_log.mul_(0.5)
    m.A  # noqa: B018  made again, in its own memory
    assert torch.equal(other.A, -torch.exp(other.a_log)) and not torch.equal(other.A, m.A)


@pytest.mark.parametrize("weights_only", [True, False])
def test_a_saved_weight_is_loaded_without_copies(weights_only):
    w = block().a_log
    w.add_(0)
    mamba1._decay(w)
    w.mul_(0.5)
    file = io.BytesIO()
    torch.save(w, file)
    file.seek(0)
    loaded = torch.load(file, weights_only=weights_only)
    assert torch.equal(mamba1._decay(loaded), -torch.exp(w))


def test_data_assigned():
    """w.data = another tensor leaves the version counter where it is."""
    m = block()
    at = m.A.data_ptr()
    m.a_log.data = m.a_log.data * 0.5
    assert torch.equal(m.A, -torch.exp(m.a_log)) and m.A.data_ptr() == at
    m.a_log.data.mul_(0.5)
    step.drop_derived(m.a_log)
    assert torch.equal(m.A, -torch.exp(m.a_log))
