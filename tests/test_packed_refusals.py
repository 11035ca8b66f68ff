"""The packed, slot, layer norm and dropout calls refuse operands that do not fit
together before anything is launched (on the CPU: no kernel is reached)."""

import ctypes

import pytest
import torch

import mamba_hip
from mamba_hip import _lib
from test_abi import _c_layout

F, BF, I = torch.float32, torch.bfloat16, torch.int32
z = lambda *s, dtype=F: torch.zeros(*s, dtype=dtype)  # noqa: E731


def scan(**over):
    a = dict(u=z(10, 6), delta=z(10, 6), A=z(6, 16), B=z(10, 16), C=z(10, 16), cu_seqlens=z(3, dtype=I), D=z(6), z=z(10, 6),
             delta_bias=z(6))
    a.update(over)
    return a


SCAN = [(dict(u=z(10, 6, dtype=torch.float16)), "u"), (dict(delta=z(9, 6)), "delta"), (dict(delta=z(10, 6, dtype=BF)), "delta"),
        (dict(B=z(10, 15)), "B"), (dict(C=z(10, 32)[:, ::2]), "C"), (dict(A=z(5, 16)), "A"), (dict(A=z(6, 32)[:, ::2]), "A"),
        (dict(A=z(6, 16, dtype=BF)), "A"), (dict(cu_seqlens=z(3, dtype=torch.int64)), "cu_seqlens"), (dict(cu_seqlens=z(0, dtype=I)), "cu_seqlens"),
        (dict(cu_seqlens=z(6, dtype=I)[::2]), "cu_seqlens"), (dict(D=z(5)), "D"), (dict(z=z(10, 5)), "z"), (dict(delta_bias=z(6, 1)), "delta_bias"),
        (dict(), "GPU device")]


@pytest.mark.parametrize("over,what", SCAN)
def test_scan(over, what):
    with pytest.raises(mamba_hip.MambaHipError, match=what):
        mamba_hip.mamba1_scan_packed(**scan(**over))
    with pytest.raises(mamba_hip.MambaHipError, match=what):
        mamba_hip.mamba1_scan_packed_bwd(z(10, 6, dtype=over["u"].dtype if "u" in over else F), **scan(**over))


@pytest.mark.parametrize("over,what", [(dict(state=z(1, 6, 16)), "row per sequence"), (dict(state=z(2, 6, 15)), "state"),
                                       (dict(state=z(2, 6, 16, dtype=BF)), "state"), (dict(slots=z(2, dtype=I)), "slots"),
                                       (dict(state=z(2, 6, 16), slots=z(3, dtype=I)), "slots"),
                                       (dict(state=z(2, 6, 16), slots=z(2, dtype=torch.int64)), "slots"),
                                       (dict(y=z(10, 6, dtype=BF)), "y"), (dict(y=z(9, 6)), "y")])
def test_scan_states(over, what):
    with pytest.raises(mamba_hip.MambaHipError, match=what):
        mamba_hip.mamba1_scan_packed(**scan(**over))


def test_scan_gradient():
    with pytest.raises(mamba_hip.MambaHipError, match="dy"):
        mamba_hip.mamba1_scan_packed_bwd(z(10, 5), **scan())
    with pytest.raises(mamba_hip.MambaHipError, match="initial_state"):
        mamba_hip.mamba1_scan_packed_bwd(z(10, 6), **scan(), initial_state=z(3, 6, 16))
    with pytest.raises(mamba_hip.MambaHipError, match="d_final_state"):
        mamba_hip.mamba1_scan_packed_bwd(z(10, 6), **scan(), d_final_state=z(2, 6, 15))
    with pytest.raises(mamba_hip.MambaHipError, match="initial_state"):
        mamba_hip.mamba1_scan_packed_autograd(**scan(), initial_state=z(2, 6, 15))


CONV = [(dict(x=z(10, 6, dtype=torch.float16)), "x"), (dict(w=z(5, 4)), "w"), (dict(w=z(6, 4, dtype=BF)), "w"), (dict(bias=z(5)), "bias"),
        (dict(x=z(10, 12)[:, ::2]), "x"), (dict(cu_seqlens=z(3)), "cu_seqlens"), (dict(), "GPU device")]


@pytest.mark.parametrize("over,what", CONV)
def test_conv(over, what):
    a = dict(x=z(10, 6), w=z(6, 4), cu_seqlens=z(3, dtype=I), bias=z(6))
    a.update(over)
    with pytest.raises(mamba_hip.MambaHipError, match=what):
        mamba_hip.conv1d_packed(**a)
    with pytest.raises(mamba_hip.MambaHipError, match=what):
        mamba_hip.conv1d_packed_bwd(z(10, 6, dtype=a["x"].dtype), **a)


def test_conv_states():
    a = dict(x=z(10, 6), w=z(6, 4), cu_seqlens=z(3, dtype=I))
    for over, what in ((dict(state=z(2, 6, 3)), "state"), (dict(state=z(1, 6, 4)), "row per sequence"), (dict(out=z(10, 5)), "out")):
        with pytest.raises(mamba_hip.MambaHipError, match=what):
            mamba_hip.conv1d_packed(**a, **over)


def test_steps():
    for over, what in ((dict(state=z(2, 6, 4)), "row per sequence"), (dict(slots=z(2, dtype=I)), "slots"), (dict(out=z(3, 5)), "out"),
                       (dict(), "GPU device")):
        a = dict(x=z(3, 6), state=z(3, 6, 4), slots=None, w=z(6, 4))
        a.update(over)
        with pytest.raises(mamba_hip.MambaHipError, match=what):
            mamba_hip.conv1d_step_slots(**a)
    for over, what in ((dict(state=z(2, 6, 16)), "row per sequence"), (dict(B=z(3, 15)), "B"), (dict(z=z(3, 6, dtype=BF)), "z"),
                       (dict(), "GPU device")):
        a = dict(u=z(3, 6), delta=z(3, 6), A=z(6, 16), B=z(3, 16), C=z(3, 16), state=z(3, 6, 16), slots=None)
        a.update(over)
        with pytest.raises(mamba_hip.MambaHipError, match=what):
            mamba_hip.scan_step_slots(**a)


def test_layer_norm():
    for a, what in ((dict(x=z(4, 8, dtype=torch.float16), weight=z(8)), "x"), (dict(x=z(4, 8), weight=z(7)), "weight"),
                    (dict(x=z(4, 8), weight=z(8), bias=z(8, dtype=BF)), "bias"), (dict(x=z(4, 8), weight=z(8), eps=-1.0), "eps"),
                    (dict(x=z(4, 0), weight=z(0)), "x"), (dict(x=z(4, 8), weight=z(8), stats=(z(3), z(4))), "mean"),
                    (dict(x=z(4, 8), weight=z(8)), "GPU device")):
        with pytest.raises(mamba_hip.MambaHipError, match=what):
            mamba_hip.layer_norm(**a)
    for a, what in ((dict(dy=z(3, 8)), "dy"), (dict(dy=z(4, 8, dtype=BF)), "dy"), (dict(mean=z(3)), "mean"), (dict(rstd=None), "rstd")):
        b = dict(dy=z(4, 8), x=z(4, 8), weight=z(8), mean=z(4), rstd=z(4))
        b.update(a)
        with pytest.raises(mamba_hip.MambaHipError, match=what):
            mamba_hip.layer_norm_bwd(**b)


def test_dropout():
    rng = z(2, dtype=torch.int64)
    for a, what in ((dict(x=z(4, dtype=torch.float16)), "x"), (dict(p=1.5), "p"), (dict(p=float("nan")), "p"), (dict(rng=z(2)), "rng"),
                    (dict(rng=z(3, dtype=torch.int64)), "rng"), (dict(residual=z(5)), "residual"), (dict(out=z(4, dtype=BF)), "out"),
                    (dict(), "GPU device")):
        b = dict(x=z(4), p=0.5, rng=rng)
        b.update(a)
        with pytest.raises(mamba_hip.MambaHipError, match=what):
            mamba_hip.dropout(**b)


def test_the_library_refuses_by_itself():
    """Status codes without a GPU: every pointer is checked before a launch."""
    L, P = _lib.lib(), 4096  # never dereferenced
    a = _lib.Mamba1ScanPackedArgs()
    assert L.mamba1_scan_packed_fwd(None, None, 0, None) == 1
    a.rows, a.nseq, a.dim, a.dstate = 300, 2, 8, 65
    assert L.mamba1_scan_packed_fwd(ctypes.byref(a), None, 0, None) == 2 and b"dstate" in L.mamba_last_error()
    a.dstate = 16
    assert L.mamba1_scan_packed_fwd(ctypes.byref(a), None, 0, None) == 1
    for k in ("cu_seqlens", "u", "delta", "A", "B", "C", "y"):
        setattr(a, k, P)
    assert L.mamba1_scan_packed_fwd(ctypes.byref(a), None, 0, None) == 1 and b"overlap" in L.mamba_last_error()
    b = _lib.Mamba1ScanPackedBwdArgs()
    b.fwd = a
    assert L.mamba1_scan_packed_bwd(ctypes.byref(b), None, 0, None) == 1 and b"dA" in L.mamba_last_error()
    for i, k in enumerate(("dA", "dy", "du", "ddelta", "dB", "dC")):
        setattr(b, k, P + (i + 1) * 300 * 64 * 4)
    for k in ("du_st", "ddelta_st", "dB_st", "dC_st"):
        setattr(b, k, 64)
    need = L.mamba1_scan_packed_bwd_workspace_size(ctypes.byref(b))
    assert need > 0
    assert L.mamba1_scan_packed_bwd(ctypes.byref(b), ctypes.c_void_p(P), need - 1, None) == 3
    assert L.mamba1_scan_packed_bwd(ctypes.byref(b), ctypes.c_void_p(P + 4), need, None) == 1
    b.fwd.z = P
    assert L.mamba1_scan_packed_bwd(ctypes.byref(b), ctypes.c_void_p(P), need, None) == 1 and b"dz" in L.mamba_last_error()
    c = _lib.Conv1dPackedArgs()
    c.rows, c.nseq, c.channels, c.kernel, c.w, c.cu_seqlens = 10, 1, 4, 65, P, P
    assert L.mamba_conv1d_packed_fwd(ctypes.byref(c), None) == 1 and b"kernel" in L.mamba_last_error()
    c.kernel, c.x, c.out, c.out_st, c.state, c.nslots = 4, P, P, 4, P, 0
    assert L.mamba_conv1d_packed_fwd(ctypes.byref(c), None) == 1 and b"row per sequence" in L.mamba_last_error()
    assert L.mamba_conv1d_packed_bwd(ctypes.byref(c), None, 0, None) == 1 and b"window" in L.mamba_last_error()
    n = _lib.LayerNormArgs()
    n.rows, n.cols, n.x, n.y, n.y_sr = 4, 8, P, P, 7
    assert L.mamba_layernorm_fwd(ctypes.byref(n), None) == 1 and b"overlap" in L.mamba_last_error()
    m = _lib.LayerNormBwdArgs()
    m.rows, m.cols, m.dweight = 4, 8, P
    assert L.mamba_layernorm_bwd(ctypes.byref(m), None, 0, None) == 1
    for k in ("x", "dy", "mean", "rstd"):
        setattr(m, k, P)
    assert L.mamba_layernorm_bwd(ctypes.byref(m), None, 0, None) == 3
    o = _lib.DropoutArgs()
    o.rows, o.cols, o.p = 1, 8, 1.5
    assert L.mamba_dropout(ctypes.byref(o), None) == 1
    o.p = 0.5
    assert L.mamba_dropout(ctypes.byref(o), None) == 1 and b"rng" in L.mamba_last_error()


def test_many_sequences_and_many_rows():
    """A bound on the lengths never refuses what is taken without one (here: up to the
    missing workspace), and the rows that the gradients cannot take the forward can."""
    L, P = _lib.lib(), 1 << 20  # never dereferenced
    a = _lib.Mamba1ScanPackedArgs()
    a.rows, a.nseq, a.dim, a.dstate = 10_000_000, 3_000_000, 512, 16
    for i, k in enumerate(("cu_seqlens", "u", "delta", "A", "B", "C", "y")):
        setattr(a, k, P << (20 + i))
    for k in ("u_st", "delta_st", "B_st", "C_st", "y_st"):
        setattr(a, k, 512)
    for most in (0, 10, 10_000_000):
        a.max_seqlen = most
        assert L.mamba1_scan_packed_workspace_size(ctypes.byref(a)) > 0
        assert L.mamba1_scan_packed_fwd(ctypes.byref(a), None, 0, None) == 3
    a.max_seqlen, a.rows, a.dim = 0, 40_000_000, 64
    assert L.mamba1_scan_packed_fwd(ctypes.byref(a), None, 0, None) == 3
    b = _lib.Mamba1ScanPackedBwdArgs()
    b.fwd = a
    for i, k in enumerate(("dA", "dy", "du", "ddelta", "dB", "dC")):
        setattr(b, k, P << (30 + i))
    for k in ("dy_st", "du_st", "ddelta_st", "dB_st", "dC_st"):
        setattr(b, k, 64)
    assert L.mamba1_scan_packed_bwd(ctypes.byref(b), None, 0, None) == 2 and b"too large" in L.mamba_last_error()


def test_the_library_refuses_outputs_on_inputs():
    """An output that shares memory with an input: refused but where a thread reads what it
    writes.  The workspace's absence tells that the rest was taken."""
    L, P = _lib.lib(), 1 << 20  # never dereferenced
    a = _lib.Mamba1ScanPackedArgs()
    a.rows, a.nseq, a.dim, a.dstate = 300, 2, 64, 16
    for i, k in enumerate(("cu_seqlens", "u", "delta", "A", "B", "C", "z")):
        setattr(a, k, P * (i + 1))
    for k in ("u_st", "delta_st", "z_st", "B_st", "C_st"):
        setattr(a, k, 128)
    scan = lambda y, st: (setattr(a, "y", y), setattr(a, "y_st", st), L.mamba1_scan_packed_fwd(ctypes.byref(a), None, 0, None))[2]  # noqa: E731
    for ok in ((9 * P, 64), (a.u, 128), (a.z, 128), (a.delta, 128), (a.u + 64 * 4, 128), (a.B + 16 * 4, 128), (a.C + 64 * 4, 128)):
        assert scan(*ok) == 3, ok
    for bad in ((a.u, 64), (a.u + 4, 128), (a.u + 128 * 4, 128), (a.z - 63 * 4, 128), (a.B, 128), (a.B + 15 * 4, 128), (a.C - 4, 128),
                (a.C + 300 * 128 * 4 - 112 * 4 - 4, 128)):
        assert scan(*bad) == 1 and b"overlaps" in L.mamba_last_error(), bad
    c = _lib.Conv1dPackedArgs()
    c.rows, c.nseq, c.channels, c.kernel, c.w, c.cu_seqlens, c.x, c.x_st = 10, 1, 4, 4, P, 2 * P, 3 * P, 8
    for out, st in ((3 * P, 8), (3 * P + 12, 8), (3 * P - 4, 4)):
        c.out, c.out_st = out, st
        assert L.mamba_conv1d_packed_fwd(ctypes.byref(c), None) == 1 and b"overlaps" in L.mamba_last_error()
    n = _lib.LayerNormArgs()
    n.rows, n.cols, n.x, n.x_sr, n.y, n.y_sr = 4, 8, P, 8, P + 4, 8
    assert L.mamba_layernorm_fwd(ctypes.byref(n), None) == 1 and b"overlaps" in L.mamba_last_error()
    o = _lib.DropoutArgs()
    o.rows, o.cols, o.p, o.rng, o.x, o.residual, o.out = 1, 8, 0.5, P, 2 * P, 3 * P, 3 * P + 4
    assert L.mamba_dropout(ctypes.byref(o), None) == 1 and b"overlaps" in L.mamba_last_error()
    g = _lib.Mamba1ScanPackedBwdArgs()
    g.fwd, outs = a, ("du", "ddelta", "dz", "dB", "dC")
    g.dA, g.dy, g.dy_st = P, 19 * P, 128
    for i, k in enumerate(outs):
        setattr(g, k, P * (20 + i))
        setattr(g, k + "_st", 128)
    bwd = lambda: L.mamba1_scan_packed_bwd(ctypes.byref(g), None, 0, None)  # noqa: E731
    assert bwd() == 3
    for k in outs:
        mine = getattr(g, k)
        for on in (a.u, a.z, g.dy, a.C + 4, P * 20 if k != "du" else P * 22):
            setattr(g, k, on)
            assert bwd() == 1 and b"overlap" in L.mamba_last_error(), (k, on)
        setattr(g, k, mine)
    c.dout, c.dout_st, c.dx, c.dx_st = 4 * P, 8, 4 * P, 8
    assert L.mamba_conv1d_packed_bwd(ctypes.byref(c), None, 0, None) == 1 and b"overlaps" in L.mamba_last_error()
    b = _lib.LayerNormBwdArgs()
    b.rows, b.cols, b.x, b.x_sr, b.dy, b.dy_sr, b.mean, b.rstd, b.dx, b.dx_sr = 4, 8, P, 8, 2 * P, 8, 3 * P, 4 * P, 2 * P, 8
    assert L.mamba_layernorm_bwd(ctypes.byref(b), None, 0, None) == 1 and b"overlaps" in L.mamba_last_error()


@pytest.mark.parametrize("cls_name,c_name", [("Conv1dPackedArgs", "mamba_conv1d_packed_args"), ("Conv1dStepSlotsArgs", "mamba_conv1d_step_slots_args"),
                                             ("Mamba1ScanPackedArgs", "mamba1_scan_packed_args"),
                                             ("Mamba1ScanPackedBwdArgs", "mamba1_scan_packed_bwd_args"),
                                             ("Mamba1ScanStepSlotsArgs", "mamba1_scan_step_slots_args"),
                                             ("LayerNormArgs", "mamba_layernorm_args"), ("LayerNormBwdArgs", "mamba_layernorm_bwd_args"),
                                             ("DropoutArgs", "mamba_dropout_args")])
def test_struct_layouts_match_header(cls_name, c_name):
    cls = getattr(_lib, cls_name)
    fields = [f[0] for f in cls._fields_]
    got = _c_layout(c_name, fields)
    assert got[0] == ctypes.sizeof(cls) and got[1:] == [getattr(cls, f).offset for f in fields]
