"""Argument checks of the 8-bit KV cache's entry points that need no device."""
import ctypes

import numpy as np
import pytest

from gonn_amd import _lib


def test_create_and_null_handles():
    lib = _lib.load()
    h = ctypes.c_void_p()
    for B, H, L, D, want in ((0, 1, 64, 64, _lib.GONN_E_INVALID), (1, 0, 64, 64, _lib.GONN_E_INVALID),
                             (1, 1, 0, 64, _lib.GONN_E_INVALID), (1, 1, 64, 0, _lib.GONN_E_INVALID),
                             (1, 1, 64, 96, _lib.GONN_E_UNSUPPORTED),
                             (1 << 15, 1 << 10, 1 << 10, 64, _lib.GONN_E_UNSUPPORTED)):
        assert lib.gonn_hip_kvcache8_create(ctypes.byref(h), B, H, L, D) == want
        assert not h
    assert lib.gonn_hip_kvcache8_create(None, 1, 1, 64, 64) == _lib.GONN_E_INVALID
    b = _lib.Buf(1 << 20, 1 << 20, _lib.GONN_BF16)
    n = (ctypes.c_int * 1)(0)
    assert lib.gonn_hip_kvcache8_free(None) == 0
    assert lib.gonn_hip_kvcache8_lengths(None, n, None) == _lib.GONN_E_INVALID
    assert lib.gonn_hip_kvcache8_append(None, b, b, 1, None, None) == _lib.GONN_E_INVALID
    assert lib.gonn_hip_kvcache8_truncate(None, n, None) == _lib.GONN_E_INVALID
    assert lib.gonn_hip_kvcache8_read(None, b, b, 0, 1, None) == _lib.GONN_E_INVALID
    assert lib.gonn_hip_kvcache8_attend_workspace_bytes(None, 1, 1, 0, 0, None) == 0
    assert lib.gonn_hip_kvcache8_attend(None, b, b, 1, 1, 1.0, 0, 0, None, 0, None) == _lib.GONN_E_INVALID


def test_definition_against_torch_e4m3():
    """The tests' own rounding agrees with torch's e4m3 over every bf16 number up to 448."""
    torch = pytest.importorskip("torch")
    from tests import _cache8_ref as ref
    u = torch.arange(0, 0x43e1, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).double()
    x = torch.cat([u, -u, u.new_tensor([448.0])])
    want = x.float().to(torch.float8_e4m3fn).double()
    assert torch.equal(ref.quantised(x.view(1, -1))[0], want)
