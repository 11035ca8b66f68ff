"""Mamba-1's short convolution and selective scan over packed sequences, their
gradients, and their single-token steps on a cache addressed by slot.

Packed: the rows of several sequences one behind the other in [rows, .] tensors,
sequence s being rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1 (``cu_seqlens`` int32
on the device; sequences may be empty).  Rows outside every sequence (padding) are
left as they were in an output that the caller gives, and are zero in one that is
made here.

A cache is addressed by slot: sequence (or token) s keeps its state in row
``slots[s]`` (int32; None: row s) of the cache tensor, updated in place.  The slots
of one call are distinct; one out of range is no state (zero at the start, nothing
kept).  A slot's row is zeroed by the caller before its first sequence.

Reference: ``Mamba1::forward`` layer 2 (src/mamba1/mamba1.rs:300-340),
``Mamba1::selective_scan`` (mamba1.rs:422-523), ``Mamba1::step``
(mamba1.rs:533-733), which take sequences of one length and a cache row for each.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import (Conv1dPackedArgs, Conv1dStepSlotsArgs, Mamba1ScanPackedArgs, Mamba1ScanPackedBwdArgs,
                   Mamba1ScanStepSlotsArgs, check)
from .ssd import _dtype_code, workspace


def _fail(msg: str):
    raise _lib.MambaHipError(msg)


# The checks run on every call of a step: they build a message only to raise it.

def _need(ok: bool, msg: str):
    if not ok:
        _fail(msg)


def _rows(t: torch.Tensor, name: str, rows: Optional[int] = None, cols: Optional[int] = None, dtype=None):
    """A [rows, cols] tensor whose last axis is contiguous."""
    shape = t.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (cols is not None and shape[1] != cols):
        _fail(f"{name}: shape {tuple(shape)}, expected [{'rows' if rows is None else rows}, {'cols' if cols is None else cols}]")
    if t.dtype != dtype if dtype is not None else t.dtype not in _IO:
        _fail(f"{name}: dtype {t.dtype}, expected {dtype or 'float32 or bfloat16'}")
    if t.stride(1) != 1 and shape[1] > 1:
        _fail(f"{name}: the last axis must be contiguous")


_IO = (torch.float32, torch.bfloat16)


def _param(t: Optional[torch.Tensor], name: str, *shape: int):
    if t is not None and (t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous()):
        _fail(f"{name} must be a contiguous float32 tensor of shape {shape}")


def _sequences(cu_seqlens: torch.Tensor, slots: Optional[torch.Tensor], state: Optional[torch.Tensor], name: str, *tail: int) -> int:
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or not cu_seqlens.is_contiguous():
        _fail("cu_seqlens must be a contiguous int32 tensor of one more entry than sequences")
    n = cu_seqlens.numel() - 1
    if state is not None or slots is not None:
        _slots(n, slots, state, name, *tail)
    return n


def _slots(n: int, slots, state, name: str, *tail: int):
    if state is None:
        _fail("slots without a state")
    if state.dtype != torch.float32 or state.shape[1:] != tail or not state.is_contiguous():
        _fail(f"{name} must be a contiguous float32 tensor of shape (slots, {', '.join(map(str, tail))})")
    if slots is None:
        if state.shape[0] < n:
            _fail(f"{name} needs a row per sequence where no slots are given")
    elif slots.dtype != torch.int32 or slots.shape != (n,) or not slots.is_contiguous():
        _fail(f"slots must be a contiguous int32 tensor of {n} entries")


_SAME = contextlib.nullcontext()


def _one_device(first: torch.Tensor, *ts: Optional[torch.Tensor]):
    """Every operand on one GPU, which becomes the current device for the call."""
    dev = first.get_device()  # below 0: not a GPU
    if dev < 0:
        _fail("operands on one GPU device required")
    for t in ts:
        if t is not None and t.get_device() != dev:
            _fail("operands on one GPU device required")
    return _SAME if dev == torch._C._cuda_getDevice() else torch.cuda.device(dev)


def _raw_stream(t: torch.Tensor) -> int:
    """The current stream of t's device as a handle."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


# an uninitialised tensor of t's shape and type with rows one behind the other (a few us
# less than one from shape, type and device)
_new = functools.partial(torch.empty_like, memory_format=torch.contiguous_format)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _st(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.stride(0)


def _once(fn):
    """A backward that is differentiable once: autograd's guard where a graph of the gradient
    is wanted, the function itself (which that guard would slow down) where none is."""
    guarded = once_differentiable(fn)
    return staticmethod(lambda ctx, *g: guarded(ctx, *g) if torch.is_grad_enabled() else fn(ctx, *g))


def _like_rows(dy: torch.Tensor) -> torch.Tensor:
    """A gradient as the kernels read it (autograd hands on expanded ones)."""
    return dy if dy.stride(-1) == 1 or dy.shape[-1] <= 1 else dy.contiguous()


# ------------------------------------------------------------- convolution ---

def _conv_args(x, w, cu_seqlens, bias, silu, state=None, slots=None) -> Conv1dPackedArgs:
    _rows(x, "x")
    rows, c = x.shape
    _need(w.dim() == 2, "w must be [channels, kernel]")
    k = w.shape[1]
    _param(w, "w", c, k)
    _param(bias, "bias", c)
    _sequences(cu_seqlens, slots, state, "state", c, k)
    a = _conv_fill(x, w, cu_seqlens, bias, silu)
    if state is not None:
        a.state, a.nslots, a.slots = state.data_ptr(), state.shape[0], _p(slots)
    return a


def _conv_fill(x, w, cu_seqlens, bias, silu) -> Conv1dPackedArgs:
    """The arguments of operands that have been checked."""
    a = Conv1dPackedArgs()
    (rows, c), k, a.nseq = x.shape, w.shape[1], cu_seqlens.shape[0] - 1
    a.rows, a.channels, a.kernel, a.io_dtype, a.silu = rows, c, k, _dtype_code(x), int(bool(silu))
    a.cu_seqlens = cu_seqlens.data_ptr()
    a.x, a.x_st, a.w, a.bias = x.data_ptr(), x.stride(0), w.data_ptr(), _p(bias)
    return a


def conv1d_packed(x: torch.Tensor, w: torch.Tensor, cu_seqlens: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  silu: bool = True, state: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Depthwise causal convolution (+ SiLU) of packed sequences: x [rows, c] f32 or bf16,
    w [c, K], bias [c] f32 -> [rows, c] of x's type.  ``state`` [slots, c, K] f32: the
    windows (the last K inputs) that the sequences go on from, moved on in place."""
    a = _conv_args(x, w, cu_seqlens, bias, silu, state, slots)
    a.fill_outside = int(out is None)
    if out is not None:
        _rows(out, "out", x.shape[0], x.shape[1], x.dtype)
    with _one_device(x, w, cu_seqlens, bias, state, slots, out):
        if out is None:
            out = _new(x)
        a.out, a.out_st = out.data_ptr(), out.stride(0)
        check(_lib.lib().mamba_conv1d_packed_fwd(ctypes.byref(a), _raw_stream(x)), "mamba_conv1d_packed_fwd")
    return out


def conv1d_packed_bwd(dout: torch.Tensor, x: torch.Tensor, w: torch.Tensor, cu_seqlens: torch.Tensor,
                      bias: Optional[torch.Tensor] = None, silu: bool = True) -> dict:
    """Gradients of ``conv1d_packed`` without a state: dict(dx [rows, c] of x's type, zero
    outside the sequences; dw [c, K], dbias [c] f32)."""
    a = _conv_args(x, w, cu_seqlens, bias, silu)
    _rows(dout, "dout", x.shape[0], x.shape[1], x.dtype)
    with _one_device(dout, x, w, cu_seqlens, bias):
        dx, dw, dbias = _conv_bwd(a, dout, x, w, bias)
    return dict(dx=dx, dw=dw, dbias=dbias)


def _conv_bwd(a: Conv1dPackedArgs, dout, x, w, bias):
    """``conv1d_packed_bwd`` after its checks."""
    dx = _new(x)
    dw, dbias = torch.empty_like(w), None if bias is None else torch.empty_like(bias)
    a.fill_outside = 1
    a.dout, a.dout_st = dout.data_ptr(), dout.stride(0)
    a.dx, a.dx_st, a.dw, a.dbias = dx.data_ptr(), dx.stride(0), dw.data_ptr(), _p(dbias)
    L = _lib.lib()
    ref = ctypes.byref(a)
    ws = workspace(x.device, L.mamba_conv1d_packed_bwd_workspace_size(ref))
    check(L.mamba_conv1d_packed_bwd(ref, ws.data_ptr(), ws.numel(), _raw_stream(x)), "mamba_conv1d_packed_bwd")
    return dx, dw, dbias


class _Conv1dPacked(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, cu_seqlens, bias, silu):
        ctx.silu = silu
        ctx.save_for_backward(x, w, cu_seqlens, bias)
        return conv1d_packed(x, w, cu_seqlens, bias, silu)

    @_once
    def backward(ctx, dout):
        x, w, cu_seqlens, bias = ctx.saved_tensors
        dout = _like_rows(dout)
        with _one_device(dout):
            dx, dw, dbias = _conv_bwd(_conv_fill(x, w, cu_seqlens, bias, ctx.silu), dout, x, w, bias)
        return dx, dw, None, dbias, None


def conv1d_packed_autograd(x, w, cu_seqlens, bias=None, silu: bool = True) -> torch.Tensor:
    """``conv1d_packed`` as a differentiable op: gradients of x, w and bias."""
    return _Conv1dPacked.apply(x, w, cu_seqlens, bias, silu)


def conv1d_step_slots(x: torch.Tensor, state: torch.Tensor, slots: Optional[torch.Tensor], w: torch.Tensor,
                      bias: Optional[torch.Tensor] = None, silu: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``conv1d_step`` on a cache of slots: x [b, c] f32 or bf16, state [slots, c, K] f32 (in
    place), slots [b] int32.  Returns out [b, c] of x's type; a row whose slot is out of
    range is zero."""
    _rows(x, "x")
    b, c = x.shape
    _need(w.dim() == 2, "w must be [channels, kernel]")
    k = w.shape[1]
    _param(w, "w", c, k)
    _param(bias, "bias", c)
    _slots(b, slots, state, "state", c, k)
    if out is not None:
        _rows(out, "out", b, c, x.dtype)
    with _one_device(x, state, slots, w, bias, out):
        if out is None:
            out = _new(x)
        a = Conv1dStepSlotsArgs()
        a.batch, a.channels, a.kernel, a.io_dtype, a.silu = b, c, k, _dtype_code(x), int(bool(silu))
        a.x, a.x_sb, a.state, a.nslots, a.slots = x.data_ptr(), x.stride(0), state.data_ptr(), state.shape[0], _p(slots)
        a.w, a.bias, a.out, a.out_sb = w.data_ptr(), _p(bias), out.data_ptr(), out.stride(0)
        check(_lib.lib().mamba_conv1d_step_slots(ctypes.byref(a), _raw_stream(x)), "mamba_conv1d_step_slots")
    return out


# --------------------------------------------------------------------- scan ---

def _scan_operands(u, delta, A, B, C, D, z, delta_bias):
    """Checks shared by the packed scan and the step; (rows, dim, dstate)."""
    _rows(u, "u")
    rows, d = u.shape
    _need(A.dim() == 2, "A must be [dim, dstate]")
    n = A.shape[1]
    _param(A, "A", d, n)
    _rows(delta, "delta", rows, d, u.dtype)
    _rows(B, "B", rows, n, u.dtype)
    _rows(C, "C", rows, n, u.dtype)
    if z is not None:
        _rows(z, "z", rows, d, u.dtype)
    _param(D, "D", d)
    _param(delta_bias, "delta_bias", d)
    return rows, d, n


def _scan_args(u, delta, A, B, C, cu_seqlens, D, z, delta_bias, delta_softplus, max_seqlen, state=None, slots=None):
    _, d, n = _scan_operands(u, delta, A, B, C, D, z, delta_bias)
    _sequences(cu_seqlens, slots, state, "state", d, n)
    a = Mamba1ScanPackedArgs()
    _scan_fill(a, u, delta, A, B, C, cu_seqlens, D, z, delta_bias, delta_softplus, max_seqlen)
    if state is not None:
        a.state, a.nslots, a.slots = state.data_ptr(), state.shape[0], _p(slots)
    return a


def _scan_fill(a: Mamba1ScanPackedArgs, u, delta, A, B, C, cu_seqlens, D, z, delta_bias, delta_softplus, max_seqlen):
    """The arguments of operands that have been checked."""
    (a.rows, a.dim), a.dstate, a.nseq = u.shape, A.shape[1], cu_seqlens.shape[0] - 1
    a.io_dtype, a.delta_softplus, a.max_seqlen = _dtype_code(u), int(bool(delta_softplus)), int(max_seqlen)
    a.cu_seqlens = cu_seqlens.data_ptr()
    a.u, a.u_st, a.delta, a.delta_st = u.data_ptr(), u.stride(0), delta.data_ptr(), delta.stride(0)
    a.B, a.B_st, a.C, a.C_st = B.data_ptr(), B.stride(0), C.data_ptr(), C.stride(0)
    if z is not None:
        a.z, a.z_st = z.data_ptr(), z.stride(0)
    a.A, a.D, a.delta_bias = A.data_ptr(), _p(D), _p(delta_bias)


def mamba1_scan_packed(u, delta, A, B, C, cu_seqlens, D=None, z=None, delta_bias=None, delta_softplus: bool = False,
                       state: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None, max_seqlen: int = 0,
                       y: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The selective scan of packed sequences: u, delta, z [rows, d] and B, C [rows, n] f32
    or bf16 (one type, any row strides), A [d, n], D, delta_bias [d] f32, n <= 64.
    ``state`` [slots, d, n] f32 holds what the sequences start from and is overwritten
    with what they end in; None starts from zero.  ``max_seqlen``, a bound on the longest
    sequence where the caller knows one, helps to choose the schedule (0: unknown).
    Returns y [rows, d] of u's type."""
    a = _scan_args(u, delta, A, B, C, cu_seqlens, D, z, delta_bias, delta_softplus, max_seqlen, state, slots)
    a.fill_outside = int(y is None)
    if y is not None:
        _rows(y, "y", u.shape[0], u.shape[1], u.dtype)
    with _one_device(u, delta, A, B, C, cu_seqlens, D, z, delta_bias, state, slots, y):
        if y is None:
            y = _new(u)
        a.y, a.y_st = y.data_ptr(), y.stride(0)
        L = _lib.lib()
        need = L.mamba1_scan_packed_workspace_size(ctypes.byref(a))
        ws = workspace(u.device, need) if need else None
        check(L.mamba1_scan_packed_fwd(ctypes.byref(a), _p(ws), need, _raw_stream(u)), "mamba1_scan_packed_fwd")
    return y


def mamba1_scan_packed_bwd(dy, u, delta, A, B, C, cu_seqlens, D=None, z=None, delta_bias=None, delta_softplus: bool = False,
                           initial_state=None, d_final_state=None, max_seqlen: int = 0) -> dict:
    """Gradients of the packed scan from its inputs (every intermediate is found again).
    ``initial_state`` and ``d_final_state`` [sequences, d, n] f32 or None.  Returns
    dict(du, ddelta, dz, dB, dC of their tensors' type, zero outside the sequences; dA,
    dD, d_delta_bias, d_initial_state f32; None for what was not given).  The same inputs
    give the same bits.  While it runs it takes rows / 8 states, d x n f32 each (n as 8, 16, 32
    or 64), and some: 0.5 GB at 8192 x 5120 x 16."""
    a = Mamba1ScanPackedBwdArgs()
    a.fwd = _scan_args(u, delta, A, B, C, cu_seqlens, D, z, delta_bias, delta_softplus, max_seqlen)
    d, n, s = A.shape[0], A.shape[1], cu_seqlens.numel() - 1
    _rows(dy, "dy", u.shape[0], d, u.dtype)
    _param(initial_state, "initial_state", s, d, n)
    _param(d_final_state, "d_final_state", s, d, n)
    with _one_device(dy, u, delta, A, B, C, cu_seqlens, D, z, delta_bias, initial_state, d_final_state):
        return _scan_bwd(a, dy, u, delta, A, B, C, D, z, delta_bias, initial_state, d_final_state)


def _scan_bwd(a: Mamba1ScanPackedBwdArgs, dy, u, delta, A, B, C, D, z, delta_bias, initial_state, d_final_state) -> dict:
    """``mamba1_scan_packed_bwd`` after its checks."""
    out = dict(du=_new(u), ddelta=_new(delta), dz=None if z is None else _new(z), dB=_new(B), dC=_new(C), dA=_new(A),
               dD=None if D is None else _new(D), d_delta_bias=None if delta_bias is None else _new(delta_bias),
               d_initial_state=None)
    if initial_state is not None:  # an empty sequence ends in what it starts from
        out["d_initial_state"] = torch.zeros_like(initial_state) if d_final_state is None else d_final_state.clone()
    a.initial_state, a.d_final_state = _p(initial_state), _p(d_final_state)
    a.dy, a.dy_st = dy.data_ptr(), dy.stride(0)
    a.du, a.du_st, a.ddelta, a.ddelta_st = out["du"].data_ptr(), u.shape[1], out["ddelta"].data_ptr(), u.shape[1]
    a.dB, a.dB_st, a.dC, a.dC_st = out["dB"].data_ptr(), B.shape[1], out["dC"].data_ptr(), C.shape[1]
    if z is not None:
        a.dz, a.dz_st = out["dz"].data_ptr(), z.shape[1]
    a.dA, a.dD, a.d_delta_bias, a.d_initial_state = out["dA"].data_ptr(), _p(out["dD"]), _p(out["d_delta_bias"]), _p(out["d_initial_state"])
    L = _lib.lib()
    ref = ctypes.byref(a)
    ws = workspace(u.device, L.mamba1_scan_packed_bwd_workspace_size(ref))
    check(L.mamba1_scan_packed_bwd(ref, ws.data_ptr(), ws.numel(), _raw_stream(u)), "mamba1_scan_packed_bwd")
    return out


class _ScanPacked(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, cu_seqlens, D, z, delta_bias, initial_state, delta_softplus, max_seqlen):
        shape = (cu_seqlens.numel() - 1, *A.shape)
        _param(initial_state, "initial_state", *shape)
        final = torch.zeros(shape, dtype=torch.float32, device=u.device) if initial_state is None else initial_state.clone()
        y = mamba1_scan_packed(u, delta, A, B, C, cu_seqlens, D, z, delta_bias, delta_softplus, final, None, max_seqlen)
        ctx.save_for_backward(u, delta, A, B, C, cu_seqlens, D, z, delta_bias, initial_state)
        ctx.set_materialize_grads(False)
        ctx.opts = (delta_softplus, max_seqlen)
        return y, final

    @_once
    def backward(ctx, dy, dfinal):
        u, delta, A, B, C, cu_seqlens, D, z, delta_bias, h0 = ctx.saved_tensors
        if dy is None and dfinal is None:
            return (None,) * 12
        dy = torch.zeros(u.shape, dtype=u.dtype, device=u.device) if dy is None else _like_rows(dy)
        a = Mamba1ScanPackedBwdArgs()
        _scan_fill(a.fwd, u, delta, A, B, C, cu_seqlens, D, z, delta_bias, *ctx.opts)
        with _one_device(dy):
            g = _scan_bwd(a, dy, u, delta, A, B, C, D, z, delta_bias, h0, None if dfinal is None else dfinal.contiguous())
        return (g["du"], g["ddelta"], g["dA"], g["dB"], g["dC"], None, g["dD"], g["dz"], g["d_delta_bias"],
                g["d_initial_state"], None, None)


def mamba1_scan_packed_autograd(u, delta, A, B, C, cu_seqlens, D=None, z=None, delta_bias=None, delta_softplus: bool = False,
                                initial_state=None, max_seqlen: int = 0):
    """``mamba1_scan_packed`` as a differentiable op: (y, final_state [sequences, d, n]) from
    ``initial_state`` [sequences, d, n] (None: zero), with gradients of every float input."""
    return _ScanPacked.apply(u, delta, A, B, C, cu_seqlens, D, z, delta_bias, initial_state, delta_softplus, max_seqlen)


def scan_step_slots(u, delta, A, B, C, state: torch.Tensor, slots: Optional[torch.Tensor], D=None, z=None, delta_bias=None,
                    delta_softplus: bool = False, y: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``scan_step`` on a cache of slots: u, delta, z [b, d] and B, C [b, n] f32 or bf16 (one
    type), state [slots, d, n] f32 (in place), slots [b] int32.  Returns y [b, d] of u's
    type; a row whose slot is out of range is zero."""
    b, d, n = _scan_operands(u, delta, A, B, C, D, z, delta_bias)
    _slots(b, slots, state, "state", d, n)
    if y is not None:
        _rows(y, "y", b, d, u.dtype)
    with _one_device(u, delta, A, B, C, state, slots, D, z, delta_bias, y):
        if y is None:
            y = _new(u)
        a = Mamba1ScanStepSlotsArgs()
        a.batch, a.dim, a.dstate, a.io_dtype, a.delta_softplus = b, d, n, _dtype_code(u), int(bool(delta_softplus))
        a.u, a.u_sb, a.delta, a.delta_sb = u.data_ptr(), u.stride(0), delta.data_ptr(), delta.stride(0)
        a.B, a.B_sb, a.C, a.C_sb = B.data_ptr(), B.stride(0), C.data_ptr(), C.stride(0)
        a.y, a.y_sb = y.data_ptr(), y.stride(0)
        if z is not None:
            a.z, a.z_sb = z.data_ptr(), z.stride(0)
        a.A, a.D, a.delta_bias = A.data_ptr(), _p(D), _p(delta_bias)
        a.state, a.nslots, a.slots = state.data_ptr(), state.shape[0], _p(slots)
        check(_lib.lib().mamba1_scan_step_slots(ctypes.byref(a), _raw_stream(u)), "mamba1_scan_step_slots")
    return y
