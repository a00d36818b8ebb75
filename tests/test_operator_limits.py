"""Limits of the block norms and the int8 products, checked without a GPU."""
from __future__ import annotations

import ctypes
import random

import torch

import conftest  # noqa: F401
from qcc_b200 import _lib
from qcc_b200.runtime.block_norm import BlockNorm, _overlap


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


class Parameter:
    """What BlockNorm asks of a CUDA tensor."""
    requires_grad, dtype = False, torch.float32

    def __init__(self, address, length):
        self.address, self.shape = address, (length,)

    def get_device(self):
        return 0

    def dim(self):
        return 1

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.address

    def numel(self):
        return self.shape[0]


def test_a_norm_that_is_launching_keeps_its_argument():
    """Two threads share a norm: the one that finds its weight replaced leaves the other's C argument as it was."""
    norm = BlockNorm(Parameter(256, 64), eps=1e-5, kind="rms", weight_offset=1.0)
    launching = norm._for(64, 0)
    norm.weight = Parameter(512, 32)
    replaced = norm._for(32, 0)
    assert launching._obj.weight == 256 and replaced._obj.weight == 512
    assert norm._for(32, 0) is replaced
    assert abs(norm.eps - 1e-5) < 1e-12 and norm.weight_offset == 1.0 and norm.kind == "rms" and norm.hidden == 32


def test_overlap_of_rows():
    """Against the bytes themselves; rows that are certain to overlap are found, rows that are apart never refused."""
    rng = random.Random(0)
    certain = 0
    for _ in range(4000):
        extents = []
        for _ in range(2):
            size, rows = rng.randint(1, 6), rng.randint(0, 4)
            extents.append((rng.randint(0, 40), size + rng.choice([0, 0, 1, 3, 7]), size, rows))
        if rng.random() < 0.5:  # views of one wider tensor
            extents[1] = (extents[1][0], extents[0][1], min(extents[1][2], extents[0][1]), extents[0][3])
        a, b = extents
        used = [{p + i * s + k for i in range(t) for k in range(n)} for p, s, n, t in extents]
        shared = bool(used[0] & used[1])
        found = _overlap(a, b)
        assert found == _overlap(b, a)
        dense = any(t <= 1 or s == n for _, s, n, t in extents)
        if a[1] == b[1] or dense:
            assert found == shared, (a, b)
            certain += shared
        else:
            assert not found or shared
    assert certain > 300
