"""Limits of the block norms and the int8 products, checked without a GPU."""
from __future__ import annotations

import ctypes

import conftest  # noqa: F401
from qcc_b200 import _lib


def test_wait_limit_is_a_minute_at_most():
    lib = _lib.library()
    assert lib.qcc_set_wait_limit(60_000_000_001) == _lib.ERR_INVALID_ARGUMENT
    assert lib.qcc_set_wait_limit(2_000_000_000) == _lib.OK


def test_widest_rows():
    """Rows as they are may be as wide as the int8 products' columns, normed rows 32768."""
    lib, p = _lib.library(), ctypes.c_void_p(64)

    def call(hidden, norm, out_dtype, rows=0):
        return lib.qcc_norm_rows(p, hidden, _lib.DTYPE_BF16, rows, hidden, norm, p, hidden, out_dtype, p, None)

    rms = ctypes.byref(_lib.NormParams(None, None, _lib.DTYPE_F32, _lib.NORM_RMS, 0.0, 1e-6))
    none = ctypes.byref(_lib.NormParams(None, None, _lib.DTYPE_F32, _lib.NORM_NONE, 0.0, 0.0))
    for identity in (None, none):
        assert call(131071, identity, _lib.DTYPE_I8) == _lib.OK
        assert call(131072, identity, _lib.DTYPE_I8) == _lib.ERR_UNSUPPORTED
        assert call(32769, identity, _lib.DTYPE_BF16) == _lib.ERR_UNSUPPORTED
    assert call(32768, rms, _lib.DTYPE_I8) == _lib.OK
    assert call(32769, rms, _lib.DTYPE_I8) == _lib.ERR_UNSUPPORTED
