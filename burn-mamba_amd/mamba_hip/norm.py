"""Layer norm, RMS norm with the residual's addition, and dropout for a residual stack.

``layer_norm`` stands beside the reference's RmsNorm (src/modules/norm/rms_norm.rs;
``rmsnorm``) for stacks that centre their rows, with its gradients; ``add_rms_norm`` is that norm with the
sum before it, its gradients, and rows of 8 bits for the product behind it; ``dropout`` (with
the residual sum of src/modules/layer.rs:224-232) computes its mask where it is used.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from ._lib import AddRmsNormArgs, AddRmsNormBwdArgs, DropoutArgs, LayerNormArgs, LayerNormBwdArgs, check
from .packed import _IO, _fail, _need, _new, _once, _one_device, _p, _param, _raw_stream
from .ssd import _dtype_code, workspace


def _matrix(t: torch.Tensor, name: str) -> torch.Tensor:
    """t as [rows, cols] rows of its last axis, in place where its strides allow."""
    shape = t.shape
    if len(shape) < 1 or shape[-1] < 1:
        _fail(f"{name}: a last axis of at least one element required")
    if t.dtype not in _IO:
        _fail(f"{name}: dtype {t.dtype}, expected float32 or bfloat16")
    m = t if len(shape) == 2 else t.reshape(-1, shape[-1])
    return m if m.stride(1) == 1 or m.shape[1] == 1 else m.contiguous()


def _into(out: Optional[torch.Tensor], x: torch.Tensor) -> tuple:
    """The result tensor and its rows; one that is given has to be written in place."""
    if out is None:
        out = _new(x)
        return out, out if out.dim() == 2 else out.view(-1, out.shape[-1])
    _need(out.shape == x.shape and out.dtype == x.dtype, "out must match x")
    m = _matrix(out, "out")
    _need(m.data_ptr() == out.data_ptr(), "out must be rows of contiguous elements")
    return out, m


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               out: Optional[torch.Tensor] = None, stats: Optional[tuple] = None) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x (f32 or bf16; weight
    and bias [cols] f32 or None).  ``stats``: two f32 tensors of a value per row that take
    the mean and the reciprocal standard deviation, for ``layer_norm_bwd``."""
    m = _matrix(x, "x")
    mean, rstd = stats if stats is not None else (None, None)
    _param(mean, "mean", m.shape[0])
    _param(rstd, "rstd", m.shape[0])
    return _ln_fwd(m, x, weight, bias, eps, out, mean, rstd, _p(mean), _p(rstd))


def _ln_fwd(m, x, weight, bias, eps, out, mean, rstd, mean_at, rstd_at):
    """``layer_norm`` of the rows m of x, the statistics' places as pointers."""
    rows, cols = m.shape
    _param(weight, "weight", cols)
    _param(bias, "bias", cols)
    _need(eps >= 0, "eps must be >= 0")
    with _one_device(m, weight, bias, mean, rstd, out):
        out, o = _into(out, x)
        a = LayerNormArgs()
        a.rows, a.cols, a.io_dtype, a.eps = rows, cols, _dtype_code(m), float(eps)
        a.x, a.x_sr, a.weight, a.bias = m.data_ptr(), m.stride(0), _p(weight), _p(bias)
        a.y, a.y_sr, a.mean, a.rstd = o.data_ptr(), o.stride(0), mean_at, rstd_at
        check(_lib.lib().mamba_layernorm_fwd(ctypes.byref(a), _raw_stream(x)), "mamba_layernorm_fwd")
    return out


def layer_norm_bwd(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor) -> dict:
    """Gradients of ``layer_norm`` from its input and the forward's statistics: dict(dx of x's
    type, dweight and dbias [cols] f32).  The same inputs give the same bits."""
    m, g = _matrix(x, "x"), _matrix(dy, "dy")
    rows, cols = m.shape
    _need(g.shape == m.shape and g.dtype == m.dtype, "dy must match x")
    _param(weight, "weight", cols)
    _need(mean is not None and rstd is not None, "mean and rstd are required")
    _param(mean, "mean", rows)
    _param(rstd, "rstd", rows)
    with _one_device(m, g, weight, mean, rstd):
        dx, dweight, dbias = _ln_bwd(g, m, weight, mean.data_ptr(), rstd.data_ptr(), x)
    return dict(dx=dx, dweight=dweight, dbias=dbias)


def _ln_bwd(g, m, weight, mean: int, rstd: int, x):
    """``layer_norm_bwd`` after its checks (m: the rows of x), the statistics as pointers."""
    a = LayerNormBwdArgs()
    rows, cols = m.shape
    dx = _new(x)
    dweight = m.new_empty(cols, dtype=torch.float32) if weight is None else _new(weight)
    dbias = _new(dweight)
    a.rows, a.cols, a.io_dtype = rows, cols, _dtype_code(m)
    a.x, a.x_sr, a.dy, a.dy_sr = m.data_ptr(), m.stride(0), g.data_ptr(), g.stride(0)
    a.weight, a.mean, a.rstd = _p(weight), mean, rstd
    a.dx, a.dx_sr, a.dweight, a.dbias = dx.data_ptr(), cols, dweight.data_ptr(), dbias.data_ptr()
    L = _lib.lib()
    ref = ctypes.byref(a)
    ws = workspace(m.device, L.mamba_layernorm_bwd_workspace_size(ref))
    check(L.mamba_layernorm_bwd(ref, ws.data_ptr(), ws.numel(), _raw_stream(m)), "mamba_layernorm_bwd")
    return dx, dweight, dbias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        m = _matrix(x, "x")
        stats = m.new_empty((2, m.shape[0]), dtype=torch.float32)
        at = stats.data_ptr()
        y = _ln_fwd(m, x, weight, bias, eps, None, None, None, at, at + 4 * m.shape[0])
        ctx.save_for_backward(x, weight, stats)
        ctx.has_bias = bias is not None
        return y

    @_once
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        m, g, at = _matrix(x, "x"), _matrix(dy, "dy"), stats.data_ptr()
        with _one_device(g):
            dx, dweight, dbias = _ln_bwd(g, m, weight, at, at + 4 * m.shape[0], x)
        return dx, None if weight is None else dweight, dbias if ctx.has_bias else None, None


def layer_norm_autograd(x, weight, bias=None, eps: float = 1e-5) -> torch.Tensor:
    """``layer_norm`` as a differentiable op: gradients of x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, eps)


def _stream_rows(x, m, residual, residual_out):
    """The stream's rows of ``add_rms_norm``: (residual's rows, s, s's rows), None without one."""
    if residual is None:
        _need(residual_out is None, "residual_out without a residual")
        return None, None, None
    _need(residual.shape == x.shape, "residual must match x")
    _need(residual.dtype == torch.float32 or residual.dtype == x.dtype, "residual must be float32 or of x's type")
    return _matrix(residual, "residual"), *_into(residual_out, residual)


def _arn_args(x, m, weight, residual, eps, residual_out, rstd):
    """The arguments of operands on one device, and s."""
    rows, cols = m.shape
    _param(weight, "weight", cols)
    _param(rstd, "rstd", rows)
    _need(eps >= 0, "eps must be >= 0")
    res, s, sm = _stream_rows(x, m, residual, residual_out)
    a = AddRmsNormArgs()
    a.rows, a.cols, a.io_dtype, a.eps = rows, cols, _dtype_code(m), float(eps)
    a.x, a.x_sr, a.weight, a.rstd = m.data_ptr(), m.stride(0), _p(weight), _p(rstd)
    if res is None:
        a.stream_dtype = a.io_dtype
        return a, x, m
    a.stream_dtype = _dtype_code(res)
    a.residual, a.residual_sr, a.s, a.s_sr = res.data_ptr(), res.stride(0), sm.data_ptr(), sm.stride(0)
    return a, s, res


def add_rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor] = None, eps: float = 1e-5,
                 out: Optional[torch.Tensor] = None, residual_out: Optional[torch.Tensor] = None,
                 rstd: Optional[torch.Tensor] = None) -> tuple:
    """s = residual + x and y = s / sqrt(mean(s^2) + eps) * weight over the last axis: (y of x's
    type, s of residual's).  x f32 or bf16, residual float32 or of x's type (None: s is x
    itself), weight [cols] f32 or None.  ``residual_out`` may be residual itself; ``rstd``, a
    value per row in f32, takes 1 / sqrt(mean(s^2) + eps) for ``add_rms_norm_bwd``."""
    m = _matrix(x, "x")
    with _one_device(m, weight, residual, out, residual_out, rstd):
        a, s, _held = _arn_args(x, m, weight, residual, eps, residual_out, rstd)
        out, o = _into(out, x)
        a.y, a.y_sr = o.data_ptr(), o.stride(0)
        check(_lib.lib().mamba_add_rmsnorm_fwd(ctypes.byref(a), _raw_stream(x)), "mamba_add_rmsnorm_fwd")
    return out, s


_Q8 = {torch.int8: _lib.MAMBA_INT8, torch.float8_e4m3fn: _lib.MAMBA_E4M3}


def add_rms_norm_q8(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor] = None, eps: float = 1e-5,
                    dtype: torch.dtype = torch.int8, out: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                    residual_out: Optional[torch.Tensor] = None) -> tuple:
    """``add_rms_norm`` into rows of 8 bits: (q, scale, s) with y near q * scale, q int8 or
    float8_e4m3fn of x's shape and scale [rows] f32 (rows of the last axis) = max |y| / 127 or
    / 448; q is y / scale, rounded to f32 and then to the nearest code.  A row whose largest |y| is below 2^-100 has scale 0 and zeros, one with a NaN or an
    infinity in y a NaN for its scale and zeros.  Gradients do not pass it."""
    m = _matrix(x, "x")
    if dtype not in _Q8:
        _fail(f"dtype {dtype}, expected int8 or float8_e4m3fn")
    _need(out is None or (out.shape == x.shape and out.dtype == dtype and out.is_contiguous()), "out must be contiguous, of x's shape and dtype")
    _param(scale, "scale", m.shape[0])
    _need(not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual))),
          "rows of 8 bits are not differentiable: call under torch.no_grad()")
    with _one_device(m, weight, residual, out, scale, residual_out):
        a, s, _held = _arn_args(x, m, weight, residual, eps, residual_out, None)
        if out is None:
            out = _new(x, dtype=dtype)
        if scale is None:
            scale = m.new_empty(m.shape[0], dtype=torch.float32)
        a.q_dtype, a.q, a.q_sr, a.scale = _Q8[dtype], out.data_ptr(), m.shape[1], scale.data_ptr()
        check(_lib.lib().mamba_add_rmsnorm_fwd(ctypes.byref(a), _raw_stream(x)), "mamba_add_rmsnorm_fwd")
    return out, scale, s


def add_rms_norm_bwd(dy: torch.Tensor, s: torch.Tensor, weight: Optional[torch.Tensor], rstd: torch.Tensor,
                     ds: Optional[torch.Tensor] = None, x: Optional[torch.Tensor] = None) -> dict:
    """Gradients of ``add_rms_norm`` from s as it returned it, its rstd, dy and (of s, where it
    was used) ds: dict(dx of dy's type, dresidual of s's, dweight [cols] f32).  With a bf16
    stream s has been rounded; where ``x`` is given, s is the residual instead, and the sum is
    formed again.  Of one type dx and dresidual are one tensor.  The same inputs give the same
    bits."""
    m, g = _matrix(s, "s"), _matrix(dy, "dy")
    _need(g.shape == m.shape, "dy must match s")
    _need(s.dtype == torch.float32 or s.dtype == dy.dtype, "s must be float32 or of dy's type")
    _need(ds is None or (ds.shape == s.shape and ds.dtype == s.dtype), "ds must match s")
    _need(x is None or (s.dtype == torch.bfloat16 and x.shape == s.shape and x.dtype == s.dtype), "x goes with a bfloat16 residual, and must match it")
    _param(weight, "weight", m.shape[1])
    _need(rstd is not None, "rstd is required")
    _param(rstd, "rstd", m.shape[0])
    with _one_device(m, g, weight, rstd, ds, x):
        dx, dresidual, dweight = _arn_bwd(dy, g, s, m, weight, rstd, ds, x, True, True)
    return dict(dx=dx, dresidual=dresidual, dweight=dweight)


def _arn_bwd(dy, g, s, m, weight, rstd, ds, x, want_dx, want_dres):
    """``add_rms_norm_bwd`` after its checks (g, m: the rows of dy and s)."""
    a = AddRmsNormBwdArgs()
    a.rows, a.cols = m.shape
    a.io_dtype, a.stream_dtype = _dtype_code(g), _dtype_code(m)
    a.s, a.s_sr, a.dy, a.dy_sr, a.weight, a.rstd = m.data_ptr(), m.stride(0), g.data_ptr(), g.stride(0), _p(weight), rstd.data_ptr()
    d = None if ds is None else _matrix(ds, "ds")
    if d is not None:
        a.ds, a.ds_sr = d.data_ptr(), d.stride(0)
    xm = None if x is None else _matrix(x, "x")
    if xm is not None:
        a.x, a.x_sr = xm.data_ptr(), xm.stride(0)
    one = s.dtype == dy.dtype
    dres = _new(s) if want_dres or (one and want_dx) else None
    dx = dres if one else _new(dy) if want_dx else None
    dweight = m.new_empty(m.shape[1], dtype=torch.float32) if weight is None else _new(weight)
    if dres is not None:
        a.dresidual, a.dresidual_sr = dres.data_ptr(), a.cols
    if dx is not None and not one:
        a.dx, a.dx_sr = dx.data_ptr(), a.cols
    a.dweight = dweight.data_ptr()
    L = _lib.lib()
    ref = ctypes.byref(a)
    ws = workspace(m.device, L.mamba_add_rmsnorm_bwd_workspace_size(ref))
    check(L.mamba_add_rmsnorm_bwd(ref, ws.data_ptr(), ws.numel(), _raw_stream(m)), "mamba_add_rmsnorm_bwd")
    return dx, dres, dweight


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        rstd = x.new_empty(x.numel() // max(x.shape[-1], 1) if x.dim() else 1, dtype=torch.float32)
        y, s = add_rms_norm(x, weight, residual, eps, rstd=rstd)
        again = residual is not None and residual.dtype == torch.bfloat16  # s has been rounded
        ctx.save_for_backward(residual if again else s, weight, rstd, x if again else None)
        ctx.io = x.dtype
        ctx.set_materialize_grads(False)
        return (y, s) if residual is not None else y

    @_once
    def backward(ctx, dy, ds=None):
        s, weight, rstd, x = ctx.saved_tensors
        wx, ww, wr = ctx.needs_input_grad[:3]
        if dy is None:  # the sum alone was used
            if ds is None:
                return (None,) * 4
            return ds.to(ctx.io), torch.zeros_like(weight) if ww else None, ds, None
        m, g = _matrix(s, "s"), _matrix(dy, "dy")
        with _one_device(g):
            dx, dres, dweight = _arn_bwd(dy, g, s, m, weight, rstd, ds, x, wx, wr)
        return dx, dweight if ww else None, dres if wr else None, None


def add_rms_norm_autograd(x, weight, residual=None, eps: float = 1e-5) -> tuple:
    """``add_rms_norm`` as a differentiable op: (y, s), with gradients of x, weight and residual.
    The backward keeps s, or x and a bf16 residual, whose sum it forms again."""
    if residual is None:
        return _AddRmsNorm.apply(x, weight, None, eps), x
    return _AddRmsNorm.apply(x, weight, residual, eps)


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor, offset: int = 0, residual: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + (x / (1 - p) where kept, else 0), an element being kept with probability
    1 - p (x f32 or bf16; a dropped element's value is not looked at).

    ``rng``: two int64 on the device, (seed, call number).  The mask is Philox 4x32-10 at
    (element's place, rng[1] + offset) under the key rng[0]: a function of these alone, so
    the same call gives the same mask, and the gradient of x is this call on dy.  A program
    gives each of a step's calls its own ``offset`` and adds their count to rng[1] after the
    step's backward; in a captured graph rng is read at each replay."""
    if x.dtype not in _IO:
        _fail(f"x: dtype {x.dtype}, expected float32 or bfloat16")
    _need(0.0 <= p <= 1.0, "p must be in [0, 1]")
    _need(rng.dtype == torch.int64 and rng.shape == (2,) and rng.is_contiguous(), "rng must be two int64: (seed, call number)")
    _need(residual is None or (residual.shape == x.shape and residual.dtype == x.dtype), "residual must match x")
    _need(out is None or (out.shape == x.shape and out.dtype == x.dtype), "out must match x")
    with _one_device(x, rng, residual, out):
        if out is None:
            out = _new(x)
        n = x.numel()
        if n == 0:
            return out
        a = DropoutArgs()
        a.io_dtype, a.p = _dtype_code(x), p
        a.rng, a.offset = rng.data_ptr(), offset
        if x.is_contiguous() and out.is_contiguous() and (residual is None or residual.is_contiguous()):
            a.rows, a.cols, m, r = 1, n, x, residual  # one row
            a.x, a.out, a.residual = x.data_ptr(), out.data_ptr(), _p(residual)
        else:
            m, o = _matrix(x, "x"), _matrix(out, "out")
            _need(o.data_ptr() == out.data_ptr(), "out must be rows of contiguous elements")
            a.rows, a.cols = m.shape
            a.x, a.x_sr, a.out, a.out_sr = m.data_ptr(), m.stride(0), o.data_ptr(), o.stride(0)
            if residual is not None:
                r = _matrix(residual, "residual")
                a.residual, a.residual_sr = r.data_ptr(), r.stride(0)
        check(_lib.lib().mamba_dropout(ctypes.byref(a), _raw_stream(x)), "mamba_dropout")
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng, offset, residual):
        ctx.save_for_backward(rng)  # changed in place before the backward: autograd refuses
        ctx.call = (p, offset, residual is not None)
        return dropout(x, p, rng, offset, residual)

    @_once
    def backward(ctx, dy):
        (rng,), (p, offset, has_residual) = ctx.saved_tensors, ctx.call
        dx = dropout(dy, p, rng, offset) if ctx.needs_input_grad[0] else None
        return dx, None, None, None, dy if has_residual else None


def dropout_autograd(x, p: float, rng: torch.Tensor, offset: int = 0, residual=None) -> torch.Tensor:
    """``dropout`` as a differentiable op: gradients of x (the same mask, found again) and of
    the residual.  ``rng`` must keep its values until the backward has run."""
    return _Dropout.apply(x, p, rng, offset, residual)
