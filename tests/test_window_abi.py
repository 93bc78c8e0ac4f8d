"""Argument checks of the sliding-window entry points: host only, nothing is launched."""
import ctypes

import pytest

from gonn_amd import _lib

GOOD = dict(B=1, H=4, Hkv=2, Sq=40, Sk=50, D=64, window=8, sinks=2)
PTR = 1 << 20  # never read: every call here is refused


def _args(cls, dt=None, **kw):
    n = {**GOOD, **kw}
    dt = _lib.GONN_BF16 if dt is None else dt
    size = 4 if dt == _lib.GONN_F32 else 2
    qb = n["B"] * n["H"] * n["Sq"] * n["D"] * size
    kb = n["B"] * n["Hkv"] * n["Sk"] * n["D"] * size
    a = cls()
    for f, _ in cls._fields_:
        if f in ("q", "o", "dO", "dq"):
            setattr(a, f, _lib.Buf(PTR, qb, dt))
        elif f in ("k", "v", "dk", "dv"):
            setattr(a, f, _lib.Buf(PTR, kb, dt))
        elif f == "lse":
            a.lse = _lib.Buf(PTR, n["B"] * n["H"] * n["Sq"] * 4, _lib.GONN_F32)
        elif f in n:
            setattr(a, f, n[f])
    a.scale = 0.125
    return a


def _call(a):
    lib = _lib.load()
    f = lib.gonn_hip_attn_window_bwd if hasattr(a, "dq") else lib.gonn_hip_attn_window_fwd
    return f(ctypes.byref(a), None, 0, None)


@pytest.mark.parametrize("cls", [_lib.WindowFwdArgs, _lib.WindowBwdArgs])
def test_refusals(cls):
    for kw in ({"B": 0}, {"H": 0}, {"Hkv": 0}, {"Hkv": 3}, {"Sq": 0}, {"Sk": 0}, {"D": 0},
               {"window": 0}, {"window": -1}, {"sinks": -1}):
        assert _call(_args(cls, **kw)) == _lib.GONN_E_INVALID, kw
    assert _call(_args(cls, D=80)) == _lib.GONN_E_UNSUPPORTED
    assert _call(_args(cls, B=1 << 15, H=1 << 10, Hkv=1 << 10, Sq=64)) == _lib.GONN_E_UNSUPPORTED
    for f in ("q", "k", "v", "o"):
        a = _args(cls)
        getattr(a, f).ptr = None
        assert _call(a) == _lib.GONN_E_INVALID, f
        a = _args(cls)
        getattr(a, f).ptr = PTR + 2
        assert _call(a) == _lib.GONN_E_INVALID, f
        a = _args(cls)
        getattr(a, f).bytes -= 2
        assert _call(a) == _lib.GONN_E_INVALID, f
        a = _args(cls)
        getattr(a, f).dtype = _lib.GONN_F64
        assert _call(a) == _lib.GONN_E_INVALID, f
    a = _args(cls)
    a.scale = float("nan")
    assert _call(a) == _lib.GONN_E_INVALID
    a = _args(cls)
    a.lse.bytes -= 4
    assert _call(a) == _lib.GONN_E_INVALID
    a = _args(cls)
    a.kv_len = _lib.Buf(PTR, 4, _lib.GONN_F32)
    assert _call(a) == _lib.GONN_E_INVALID


def test_backward_needs_its_buffers_and_workspace():
    for f in ("lse", "dO", "dq", "dk", "dv"):
        a = _args(_lib.WindowBwdArgs)
        getattr(a, f).ptr = None
        assert _call(a) == _lib.GONN_E_INVALID, f
    a = _args(_lib.WindowBwdArgs)
    need = _lib.load().gonn_hip_attn_workspace_bytes(_lib.GONN_OP_WINDOW_BWD, ctypes.byref(a))
    assert need > GOOD["H"] * GOOD["Sq"] * 4
    assert _call(a) == _lib.GONN_E_WORKSPACE
    assert _lib.load().gonn_hip_attn_window_bwd(ctypes.byref(a), PTR, need - 1, None) == _lib.GONN_E_WORKSPACE
    assert _lib.load().gonn_hip_attn_workspace_bytes(
        _lib.GONN_OP_WINDOW_BWD, ctypes.byref(_args(_lib.WindowBwdArgs, window=0))) == 0


@pytest.mark.parametrize("cls", [_lib.WindowFwdArgs, _lib.WindowBwdArgs])
@pytest.mark.parametrize("dt", [_lib.GONN_BF16, _lib.GONN_F32])
def test_heads_past_32_bit_offsets_are_refused(cls, dt):
    one = dict(B=1, H=1, Hkv=1, D=128, window=64)
    for kw in ({"Sq": 1 << 24}, {"Sk": 1 << 24}):
        assert _call(_args(cls, dt, **one, **kw)) == _lib.GONN_E_UNSUPPORTED, kw
