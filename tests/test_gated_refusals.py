"""The gated recurrence, the norm with the residual's addition and the 4-bit products refuse
operands that do not fit together before anything is launched (on the CPU: no kernel is
reached), in Python and at the C entries."""

import ctypes

import pytest
import torch

import mamba_hip
from mamba_hip import _lib
from test_abi import _c_layout

F, BF, H, I, U8, I8 = torch.float32, torch.bfloat16, torch.float16, torch.int32, torch.uint8, torch.int8
z = lambda *s, dtype=F: torch.zeros(*s, dtype=dtype)  # noqa: E731
Err = mamba_hip.MambaHipError


def scan(**over):
    a = dict(x=z(10, 6), r=z(10, 6), i=z(10, 6), A=z(6), cu_seqlens=z(3, dtype=I), z=z(10, 6))
    a.update(over)
    return a


SCAN = [(dict(x=z(10, 6, dtype=H)), "x"), (dict(x=z(6)), "x"), (dict(r=z(9, 6)), "r"), (dict(i=z(10, 6, dtype=BF)), "i"),
        (dict(z=z(10, 5)), "z"), (dict(r=z(10, 12)[:, ::2]), "r"), (dict(A=z(5)), "A"), (dict(A=z(6, dtype=BF)), "A"),
        (dict(A=z(12)[::2]), "A"), (dict(cu_seqlens=z(3, dtype=torch.int64)), "cu_seqlens"), (dict(cu_seqlens=z(0, dtype=I)), "cu_seqlens"),
        (dict(), "GPU device")]


@pytest.mark.parametrize("over,what", SCAN)
def test_scan(over, what):
    with pytest.raises(Err, match=what):
        mamba_hip.gated_scan_packed(**scan(**over))
    with pytest.raises(Err, match=what):
        mamba_hip.gated_scan_packed_autograd(**scan(**over))
    a = scan(**over)
    with pytest.raises(Err, match=what):
        mamba_hip.gated_scan_packed_bwd(z(10, 6, dtype=a["x"].dtype), **a, carry=z(1, 6))


@pytest.mark.parametrize("over,what", [(dict(state=z(1, 6)), "row per sequence"), (dict(state=z(2, 5)), "state"), (dict(state=z(2, 6, dtype=BF)), "state"),
                                       (dict(slots=z(2, dtype=I)), "slots"), (dict(state=z(2, 6), slots=z(3, dtype=I)), "slots"),
                                       (dict(state=z(2, 6), slots=z(2, dtype=torch.int64)), "slots"), (dict(y=z(10, 6, dtype=BF)), "y"),
                                       (dict(y=z(9, 6)), "y"), (dict(carry=z(2, 6)), "carry"), (dict(carry=z(1, 6, dtype=BF)), "carry")])
def test_scan_states(over, what):
    with pytest.raises(Err, match=what):
        mamba_hip.gated_scan_packed(**scan(**over))


def test_scan_gradient():
    bwd = mamba_hip.gated_scan_packed_bwd
    for over, what in ((dict(dy=z(10, 5)), "dy"), (dict(dy=z(10, 6, dtype=BF)), "dy"), (dict(carry=None), "carry"), (dict(carry=z(2, 6)), "carry"),
                       (dict(initial_state=z(3, 6)), "initial_state"), (dict(d_final_state=z(2, 5)), "d_final_state")):
        a = dict(dy=z(10, 6), carry=z(1, 6), **scan())
        a.update(over)
        with pytest.raises(Err, match=what):
            bwd(**a)
    with pytest.raises(Err, match="initial_state"):
        mamba_hip.gated_scan_packed_autograd(**scan(), initial_state=z(2, 5))


def test_step():
    for over, what in ((dict(state=z(2, 6)), "row per sequence"), (dict(state=z(10, 5)), "state"), (dict(slots=z(2, dtype=I)), "slots"),
                       (dict(y=z(3, 5)), "y"), (dict(z=z(10, 6, dtype=BF)), "z"), (dict(A=z(5)), "A"), (dict(), "GPU device")):
        a = dict(scan(), state=z(10, 6), slots=None)
        del a["cu_seqlens"]
        a.update(over)
        with pytest.raises(Err, match=what):
            mamba_hip.gated_step_slots(**a)


NORM = [(dict(x=z(4, 8, dtype=H)), "x"), (dict(x=z(4, 0)), "x"), (dict(weight=z(7)), "weight"), (dict(weight=z(8, dtype=BF)), "weight"),
        (dict(residual=z(3, 8)), "residual"), (dict(residual=z(4, 8, dtype=BF)), "residual"), (dict(residual=None, residual_out=z(4, 8)), "residual"),
        (dict(eps=-1.0), "eps"), (dict(), "GPU device")]


@pytest.mark.parametrize("over,what", NORM)
def test_norm(over, what, monkeypatch):
    a = dict(x=z(4, 8), weight=z(8), residual=z(4, 8))
    a.update(over)
    if what != "GPU device":  # the check of the device comes first
        import mamba_hip.norm as norm
        import contextlib
        monkeypatch.setattr(norm, "_one_device", lambda *t: contextlib.nullcontext())
    for call in (mamba_hip.add_rms_norm, mamba_hip.add_rms_norm_q8):
        with pytest.raises(Err, match=what):
            call(**a)


def test_norm_outputs(monkeypatch):
    import contextlib

    import mamba_hip.norm as norm
    monkeypatch.setattr(norm, "_one_device", lambda *t: contextlib.nullcontext())
    a = dict(x=z(4, 8), weight=z(8), residual=z(4, 8))
    for over, what in ((dict(out=z(4, 7)), "out"), (dict(out=z(4, 8, dtype=BF)), "out"), (dict(out=z(4, 16)[:, ::2]), "out"),
                       (dict(residual_out=z(4, 7)), "out"), (dict(rstd=z(3)), "rstd")):
        with pytest.raises(Err, match=what):
            mamba_hip.add_rms_norm(**a, **over)
    for over, what in ((dict(dtype=U8), "dtype"), (dict(out=z(4, 8)), "out"), (dict(scale=z(3)), "scale"),
                       (dict(out=z(4, 16, dtype=I8)[:, :8]), "out")):
        with pytest.raises(Err, match=what):
            mamba_hip.add_rms_norm_q8(**a, **over)
    with pytest.raises(Err, match="not differentiable"):
        mamba_hip.add_rms_norm_q8(z(4, 8).requires_grad_(), z(8))
    for over, what in ((dict(dy=z(4, 7)), "dy"), (dict(s=z(4, 8, dtype=BF)), "s must"), (dict(ds=z(3, 8)), "ds"), (dict(ds=z(4, 8, dtype=BF)), "ds"),
                       (dict(weight=z(7)), "weight"), (dict(rstd=None), "rstd"), (dict(rstd=z(3)), "rstd"), (dict(x=z(4, 8)), "x goes"),
                       (dict(dy=z(4, 8, dtype=BF), s=z(4, 8, dtype=BF), x=z(4, 7, dtype=BF)), "x goes")):
        b = dict(dy=z(4, 8), s=z(4, 8), weight=z(8), rstd=z(4))
        b.update(over)
        with pytest.raises(Err, match=what):
            mamba_hip.add_rms_norm_bwd(**b)


def test_pack():
    codes, scale = z(128, 10, dtype=U8), z(2, 10)
    for a, what in (((z(128, 10), scale), "codes"), ((z(128, dtype=U8), scale), "codes"), ((codes, z(2, 9)), "scale"), ((codes, z(2, 10, dtype=H)), "scale"),
                    ((codes, z(3, 10)), "group"), ((codes, scale, z(2, 10)), "zero"), ((codes, scale, z(1, 10, dtype=U8)), "zero"),
                    ((codes, scale, None, 48), "group"), ((codes, scale, None, 32), "row for each"), ((z(130, 10, dtype=U8), z(3, 10)), "group"),
                    ((z(0, 10, dtype=U8), scale), "codes"), ((codes, scale), "GPU device")):
        with pytest.raises(Err, match=what):
            mamba_hip.pack_linear_q4(*a)
    for a, what in (((z(8),), "weight"), ((z(8, 8, dtype=I),), "weight"), ((z(8, 8), 16), "group"), ((z(8, 8), 64, False, H), "scale_dtype")):
        with pytest.raises(Err, match=what):
            mamba_hip.quantize_q4(*a)


def test_product():
    w = mamba_hip.PackedQ4(128, 10, 64, F, False, z(4096, dtype=U8))
    for over, what in ((dict(x=z(3, 128, dtype=H)), "x"), (dict(x=z(3, 127)), "x"), (dict(x=z(128)), "x"), (dict(x=z(3, 256)[:, ::2]), "x"),
                       (dict(x=z(3, 128, dtype=I8)), "x_scale"), (dict(x_scale=z(3)), "x_scale"), (dict(x=z(3, 128, dtype=I8), x_scale=z(2)), "x_scale"),
                       (dict(bias=z(9)), "bias"), (dict(bias=z(10, dtype=BF)), "bias"), (dict(dtype=H), "dtype"), (dict(out=z(3, 9)), "out"),
                       (dict(out=z(3, 10), dtype=BF), "out"), (dict(out=z(3, 20)[:, ::2]), "out"), (dict(x=z(3, 128).requires_grad_()), "differentiable"),
                       (dict(), "GPU device")):
        a = dict(x=z(3, 128), weight=w)
        a.update(over)
        with pytest.raises(Err, match=what):
            mamba_hip.linear_q4(**a)


STRUCTS = {"mamba_gated_scan_args": _lib.GatedScanArgs, "mamba_gated_scan_bwd_args": _lib.GatedScanBwdArgs,
           "mamba_gated_step_slots_args": _lib.GatedStepSlotsArgs, "mamba_add_rmsnorm_args": _lib.AddRmsNormArgs,
           "mamba_add_rmsnorm_bwd_args": _lib.AddRmsNormBwdArgs, "mamba_q4_weight": _lib.Q4Weight, "mamba_linear_q4_args": _lib.LinearQ4Args}


@pytest.mark.parametrize("name", STRUCTS)
def test_struct_layouts(name):
    cls = STRUCTS[name]
    size, *offsets = _c_layout(name, [f[0] for f in cls._fields_])
    assert ctypes.sizeof(cls) == size
    assert [getattr(cls, f[0]).offset for f in cls._fields_] == offsets


P = 1 << 20  # stands for a tensor; refused before it is followed
FAR = 1 << 30


def _scan_c():
    a = _lib.GatedScanArgs()
    a.rows, a.nseq, a.dim, a.cu_seqlens, a.A = 100, 2, 64, P, P
    for k, (name, st) in enumerate((("x", "x_st"), ("r", "r_st"), ("i", "i_st"), ("z", "z_st"))):
        setattr(a, name, FAR + (k << 24))
        setattr(a, st, 64)
    a.y, a.y_st = FAR << 1, 64
    return a


def test_c_scan():
    L = _lib.lib()
    for field, bad, what in (("rows", -1, b"rows"), ("rows", 1 << 31, b"rows"), ("nseq", -1, b"nseq"), ("dim", 0, b"dim"), ("dim", (1 << 20) + 1, b"dim"),
                             ("io_dtype", 2, b"io_dtype"), ("A", None, b"A and cu_seqlens"), ("cu_seqlens", None, b"A and cu_seqlens"),
                             ("r", None, b"x, r and i"), ("y", None, b"y is"), ("y_st", 63, b"rows of y"), ("y", FAR + 4, b"overlaps"),
                             ("y", FAR + (3 << 24) + 128, b"overlaps"), ("x_st", 1 << 25, b"strides"), ("r_st", -64, b"strides"),
                             ("i_st", 1 << 40, b"strides"), ("z_st", 1 << 25, b"strides"), ("y_st", 1 << 25, b"2^25")):
        a = _scan_c()
        setattr(a, field, bad)
        assert L.mamba_gated_scan_fwd(ctypes.byref(a), None, 0, None) == 1 and what in L.mamba_last_error(), field
    assert L.mamba_gated_scan_fwd(None, None, 0, None) == 1
    a = _scan_c()
    a.state, a.nslots = P, 1
    assert L.mamba_gated_scan_fwd(ctypes.byref(a), None, 0, None) == 1 and b"row per sequence" in L.mamba_last_error()
    a = _scan_c()
    a.rows = 0
    assert L.mamba_gated_scan_fwd(ctypes.byref(a), None, 0, None) == 0  # nothing to do


def _bwd_c():
    b = _lib.GatedScanBwdArgs()
    b.fwd = _scan_c()
    b.fwd.carry, b.dy, b.dy_st, b.dA = P, FAR + (5 << 24), 64, P
    for k, n in enumerate(("dx", "dr", "di", "dz")):
        setattr(b, n, (FAR << 2) + (k << 24))
        setattr(b, n + "_st", 64)
    return b


def test_c_scan_bwd():
    L = _lib.lib()
    for field, bad, what in (("dA", None, b"dA"), ("dy", None, b"carry, dy"), ("dz", None, b"dz goes with z"), ("dx_st", 60, b"overlap"),
                             ("dx", FAR, b"overlaps an input"), ("dr", (FAR << 2) + 64, b"two gradients"), ("di", FAR + (5 << 24), b"overlaps an input"),
                             ("dy_st", 1 << 25, b"strides"), ("dy_st", -1, b"strides"), ("dz_st", 1 << 25, b"2^25")):
        b = _bwd_c()
        setattr(b, field, bad)
        assert L.mamba_gated_scan_bwd(ctypes.byref(b), None, 0, None) == 1 and what in L.mamba_last_error(), field
    b = _bwd_c()
    b.fwd.carry = None
    assert L.mamba_gated_scan_bwd(ctypes.byref(b), None, 0, None) == 1 and b"carry" in L.mamba_last_error()
    b = _bwd_c()
    b.fwd.state = P
    assert L.mamba_gated_scan_bwd(ctypes.byref(b), None, 0, None) == 1 and b"initial_state" in L.mamba_last_error()
    assert L.mamba_gated_scan_bwd(None, None, 0, None) == 1


def test_c_step():
    L = _lib.lib()

    def args():
        a = _lib.GatedStepSlotsArgs()
        a.batch, a.dim, a.A, a.state, a.nslots = 4, 64, P, P, 4
        for k, n in enumerate("xriz"):
            setattr(a, n, FAR + (k << 24))
            setattr(a, n + "_sb", 64)
        a.y, a.y_sb = FAR << 1, 64
        return a

    for field, bad, what in (("batch", -1, b"batch"), ("batch", 65536, b"batch"), ("dim", 0, b"dim"), ("io_dtype", 3, b"io_dtype"), ("state", None, b"required"),
                             ("y", None, b"required"), ("nslots", 3, b"row per token"), ("y_sb", 63, b"rows of y"), ("y", FAR + 8, b"overlaps")):
        a = args()
        setattr(a, field, bad)
        assert L.mamba_gated_step_slots(ctypes.byref(a), None) == 1 and what in L.mamba_last_error(), field


def test_c_norm():
    L = _lib.lib()

    def args():
        a = _lib.AddRmsNormArgs()
        a.rows, a.cols, a.eps = 10, 64, 1e-5
        for k, (n, s) in enumerate((("x", "x_sr"), ("residual", "residual_sr"), ("s", "s_sr"), ("y", "y_sr"))):
            setattr(a, n, FAR + (k << 24))
            setattr(a, s, 64)
        return a

    for field, bad, what in (("rows", -1, b"rows"), ("cols", 0, b"cols"), ("io_dtype", 2, b"io_dtype"), ("stream_dtype", 1, b"io_dtype"), ("eps", -1.0, b"eps"),
                             ("y", None, b"one of y and q"), ("q", P, b"one of y and q"), ("x", None, b"x is"), ("s", None, b"s goes"), ("residual", None, b"s goes"),
                             ("y_sr", 63, b"overlap"), ("s_sr", 63, b"overlap"), ("y", FAR + 4, b"overlaps"), ("s", FAR + (3 << 24) + 64, b"overlaps"),
                             ("y", FAR + (1 << 24), b"overlaps")):
        a = args()
        setattr(a, field, bad)
        assert L.mamba_add_rmsnorm_fwd(ctypes.byref(a), None) == 1 and what in L.mamba_last_error(), field
    a = args()
    a.y, a.q, a.q_sr = None, P, 64
    assert L.mamba_add_rmsnorm_fwd(ctypes.byref(a), None) == 1 and b"q_dtype" in L.mamba_last_error()
    a.q_dtype = 2
    assert L.mamba_add_rmsnorm_fwd(ctypes.byref(a), None) == 1 and b"scale" in L.mamba_last_error()

    def back():
        b = _lib.AddRmsNormBwdArgs()
        b.rows, b.cols, b.rstd, b.dweight = 10, 64, P, P
        for k, n in enumerate(("s", "dy", "ds", "dx", "dresidual")):
            setattr(b, n, FAR + (k << 24))
            setattr(b, n + "_sr", 64)
        return b

    for field, bad, what in (("rstd", None, b"required"), ("dy", None, b"required"), ("dx_sr", 63, b"overlap"), ("dx", FAR, b"overlaps an input"),
                             ("dresidual", FAR + (3 << 24) + 64, b"dresidual"), ("stream_dtype", 1, b"io_dtype"),
                             ("x", FAR + (5 << 24), b"bf16 stream")):
        b = back()
        setattr(b, field, bad)
        assert L.mamba_add_rmsnorm_bwd(ctypes.byref(b), P, 1 << 20, None) == 1 and what in L.mamba_last_error(), field
    b = back()
    assert L.mamba_add_rmsnorm_bwd_workspace_size(ctypes.byref(b)) > 0
    assert L.mamba_add_rmsnorm_bwd(ctypes.byref(b), None, 0, None) == 3 and b"workspace" in L.mamba_last_error()


def test_c_product():
    L = _lib.lib()

    def args():
        a = _lib.LinearQ4Args()
        a.w.d_in, a.w.d_out, a.w.group, a.w.packed = 256, 64, 64, P
        a.rows, a.x, a.x_ld, a.y, a.y_ld = 3, FAR, 256, FAR << 1, 64
        return a

    for field, bad, what in (("rows", -1, b"rows"), ("x_dtype", 3, b"x_dtype"), ("y_dtype", 2, b"y_dtype"), ("x_dtype", 2, b"x_scale"), ("x_scale", P, b"x_scale"),
                             ("x", None, b"required"), ("y", None, b"required"), ("y_ld", 63, b"rows of y"), ("y", FAR + 64, b"overlaps")):
        a = args()
        setattr(a, field, bad)
        assert L.mamba_linear_q4_fwd(ctypes.byref(a), None, 0, None) == 1 and what in L.mamba_last_error(), field
    for field, bad in (("d_in", 0), ("d_out", 0), ("d_in", (1 << 22) + 1), ("group", 16), ("group", 0), ("scale_dtype", 2)):
        a = args()
        setattr(a.w, field, bad)
        assert L.mamba_linear_q4_fwd(ctypes.byref(a), None, 0, None) == 1 and b"group 32" in L.mamba_last_error(), field
        assert L.mamba_linear_q4_packed_size(ctypes.byref(a.w)) == 0
        assert L.mamba_linear_q4_pack(ctypes.byref(a.w), P, P, None, P, None) == 1
    a = args()
    a.w.packed = P + 4
    assert L.mamba_linear_q4_fwd(ctypes.byref(a), None, 0, None) == 1 and b"aligned" in L.mamba_last_error()
    a = args()
    assert L.mamba_linear_q4_pack(ctypes.byref(a.w), P, P, None, None, None) == 1
    a.w.has_zero = 1
    assert L.mamba_linear_q4_pack(ctypes.byref(a.w), P, P, None, P, None) == 1 and b"zero" in L.mamba_last_error()
    # 2 blocks of k, 4 column tiles: codes, and a word for each group's scale and zero point
    assert L.mamba_linear_q4_packed_size(ctypes.byref(a.w)) == 4 * 2 * 1024 + 4 * 4 * 16 * 8
    a.w.scale_dtype = 1
    assert L.mamba_linear_q4_packed_size(ctypes.byref(a.w)) == 4 * 2 * 1024 + 4 * 4 * 16 * 4
