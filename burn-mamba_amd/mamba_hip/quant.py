"""Products of few rows with weights of 4 bits (beside ``linear``, burn::nn::Linear::forward
in the decode steps): codes of 0 to 15 with a scale, and where there are any a zero point,
for each group of input rows and output column.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from ._lib import LinearQ4Args, Q4Weight, check
from .packed import _fail, _need, _one_device, _p, _param, _raw_stream
from .ssd import _dtype_code, workspace


@dataclass(frozen=True)
class PackedQ4:
    """A [d_in, d_out] weight of 4 bits as ``linear_q4`` reads it (``pack_linear_q4``)."""
    d_in: int
    d_out: int
    group: int
    scale_dtype: torch.dtype
    has_zero: bool
    data: torch.Tensor  # uint8: codes, scales and zero points

    def _fill(self, w: Q4Weight):
        w.d_in, w.d_out, w.group, w.has_zero = self.d_in, self.d_out, self.group, self.has_zero
        w.scale_dtype = _lib.MAMBA_BF16 if self.scale_dtype == torch.bfloat16 else _lib.MAMBA_F32
        w.packed = self.data.data_ptr()


def quantize_q4(weight: torch.Tensor, group: int = 64, zero_points: bool = False, scale_dtype: torch.dtype = torch.float32) -> tuple:
    """The codes nearest to a Linear weight [d_in, d_out]: (codes [d_in, d_out] uint8, scale
    [ceil(d_in / group), d_out] of scale_dtype, zero uint8 of that shape or None), so that weight
    is near (codes - zero) * scale (zero 8 where None).  Without zero points a group's scale is
    max |w| / 7; with them its 15 steps reach from its lowest value (or 0) to its highest (or 0)."""
    _need(weight.dim() == 2 and weight.is_floating_point() and weight.numel() > 0, "weight must be a floating [d_in, d_out] tensor")
    _need(group in (32, 64, 128), "group must be 32, 64 or 128")
    _need(scale_dtype in (torch.float32, torch.bfloat16), "scale_dtype must be float32 or bfloat16")
    d_in, d_out = weight.shape
    n = -(-d_in // group)
    w = torch.zeros(n * group, d_out, dtype=torch.float32, device=weight.device)
    w[:d_in] = weight.detach()
    w = w.view(n, group, d_out)
    if zero_points:
        lo, hi = w.amin(1).clamp(max=0), w.amax(1).clamp(min=0)
        scale = (hi - lo) / 15
    else:
        scale = w.abs().amax(1) / 7
    scale = scale.to(scale_dtype)
    step = scale.float()[:, None]
    step = torch.where(step > 0, step, torch.ones_like(step))  # a group of zeros: any step
    zero = torch.round(-lo / step[:, 0]).clamp(0, 15) if zero_points else None
    codes = torch.round(w / step) + (8 if zero is None else zero[:, None])
    codes = codes.clamp(0, 15).to(torch.uint8).view(n * group, d_out)[:d_in]
    return codes.contiguous(), scale, None if zero is None else zero.to(torch.uint8)


def pack_linear_q4(codes: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor] = None, group: Optional[int] = None) -> PackedQ4:
    """Lay a weight of 4 bits out for ``linear_q4``, once, at model load: codes [d_in, d_out]
    uint8 of 0 to 15 (the low four bits are taken), scale [groups, d_out] f32 or bf16, zero
    [groups, d_out] uint8 of 0 to 16 or None (8 everywhere).  ``group``, the rows that share a scale, is
    32, 64 or 128; None: d_in / groups, where that is whole."""
    _need(codes.dim() == 2 and codes.dtype == torch.uint8 and codes.numel() > 0, "codes must be a uint8 [d_in, d_out] tensor")
    d_in, d_out = codes.shape
    _need(scale.dim() == 2 and scale.dtype in (torch.float32, torch.bfloat16) and scale.shape[1] == d_out, "scale must be float32 or bfloat16 [groups, d_out]")
    if group is None:
        group = d_in // scale.shape[0] if scale.shape[0] and d_in % scale.shape[0] == 0 else 0
    _need(group in (32, 64, 128), "group must be 32, 64 or 128")
    _need(scale.shape[0] == -(-d_in // group), "scale must have a row for each group")
    _need(zero is None or (zero.dtype == torch.uint8 and zero.shape == scale.shape), "zero must be uint8 and match scale")
    # read back at load; a capture cannot, and leaves it to the kernel, which makes a NaN of such a group
    if zero is not None and not (zero.is_cuda and torch.cuda.is_current_stream_capturing()):
        _need(int(zero.max()) <= 16, "zero points must be at most 16")
    with _one_device(codes, scale, zero):
        codes, scale = codes.contiguous(), scale.detach().contiguous()
        zero = None if zero is None else zero.contiguous()
        w = Q4Weight()
        w.d_in, w.d_out, w.group, w.scale_dtype, w.has_zero = d_in, d_out, group, _dtype_code(scale), zero is not None
        L = _lib.lib()
        data = torch.empty(L.mamba_linear_q4_packed_size(ctypes.byref(w)), dtype=torch.uint8, device=codes.device)
        check(L.mamba_linear_q4_pack(ctypes.byref(w), codes.data_ptr(), scale.data_ptr(), _p(zero), data.data_ptr(), _raw_stream(codes)),
              "mamba_linear_q4_pack")
    return PackedQ4(d_in, d_out, group, scale.dtype, zero is not None, data)


_X = {torch.float32: _lib.MAMBA_F32, torch.bfloat16: _lib.MAMBA_BF16, torch.int8: _lib.MAMBA_INT8}


def linear_q4(x: torch.Tensor, weight: PackedQ4, bias: Optional[torch.Tensor] = None, x_scale: Optional[torch.Tensor] = None,
              dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = x W + bias for few rows: x [rows, d_in] bf16, f32 or, with x_scale [rows] f32 (the rows
    of ``add_rms_norm_q8``), int8; bias [d_out] f32.  Returns [rows, d_out] of ``dtype`` (f32
    or bf16; None: x's, bf16 for int8) or in ``out``.  Sums are f32, of int8 rows exact
    within a group; a row of x with a NaN or an infinity gives a row of NaN, and values
    from 2^115 on, where sums of 31 |x| may pass f32, may.  Gradients do not pass it."""
    if x.dtype not in _X:
        _fail(f"x: dtype {x.dtype}, expected float32, bfloat16 or int8")
    _need(x.dim() == 2 and x.shape[1] == weight.d_in, "x must be [rows, d_in]")
    _need(x.stride(1) == 1 or x.shape[1] == 1, "x: the last axis must be contiguous")
    _need((x_scale is not None) == (x.dtype == torch.int8), "x_scale goes with rows of int8")
    rows = x.shape[0]
    _param(x_scale, "x_scale", rows)
    _param(bias, "bias", weight.d_out)
    _need(not (torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad))),
          "products with weights of 4 bits are not differentiable: call under torch.no_grad()")
    if out is None:
        dtype = dtype or (torch.bfloat16 if x.dtype == torch.int8 else x.dtype)
        _need(dtype in (torch.float32, torch.bfloat16), "dtype must be float32 or bfloat16")
    else:
        _need(out.shape == (rows, weight.d_out) and (dtype is None or out.dtype == dtype) and (out.stride(1) == 1 or out.shape[1] == 1),
              "out must be [rows, d_out] with a contiguous last axis")
    with _one_device(x, weight.data, bias, x_scale, out):
        if out is None:
            out = torch.empty((rows, weight.d_out), dtype=dtype, device=x.device)
        a = LinearQ4Args()
        weight._fill(a.w)
        a.rows, a.x_dtype, a.y_dtype = rows, _X[x.dtype], _dtype_code(out)
        a.x, a.x_ld, a.x_scale, a.bias = x.data_ptr(), x.stride(0), _p(x_scale), _p(bias)
        a.y, a.y_ld = out.data_ptr(), out.stride(0)
        L = _lib.lib()
        ref = ctypes.byref(a)
        need = L.mamba_linear_q4_workspace_size(ref)
        ws = workspace(x.device, need) if need else None
        check(L.mamba_linear_q4_fwd(ref, _p(ws), need, _raw_stream(x)), "mamba_linear_q4_fwd")
    return out
