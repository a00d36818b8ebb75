"""Limits of the block norms and the int8 products, checked without a GPU."""
from __future__ import annotations

import conftest  # noqa: F401
from qcc_b200 import _lib


def test_wait_limit_is_a_minute_at_most():
    lib = _lib.library()
    assert lib.qcc_set_wait_limit(60_000_000_001) == _lib.ERR_INVALID_ARGUMENT
    assert lib.qcc_set_wait_limit(2_000_000_000) == _lib.OK
