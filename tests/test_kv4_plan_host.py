"""The launch plan of kv4_attention where no GPU is needed: what it refuses before any device work."""

import ctypes as C

import pytest

import rldx_b200  # noqa: F401
from rldx_b200 import _lib


@pytest.mark.parametrize("q_heads,kv_heads,max_new,width,rc", [
    (24, 24, 1, 1 << 20, _lib.RLDX_OK),
    (24, 24, 1, (1 << 30) // 24 - 12, _lib.RLDX_OK),  # the last that one launch can count for one sequence
    (24, 24, 1, (1 << 30) // 24 - 11, _lib.RLDX_ERR_UNSUPPORTED),
    (16, 2, 4, (1 << 26) - 1, _lib.RLDX_OK),
    (64, 4, 2, (1 << 26) - 1, _lib.RLDX_OK),
    (64, 16, 5, (1 << 26) - 1, _lib.RLDX_ERR_UNSUPPORTED),
    (64, 16, 9, (1 << 26) - 1, _lib.RLDX_OK),  # more than 32 rows: the kernel for chunks counts no units
])
def test_units_that_do_not_fit_32_bits_are_refused(lib, q_heads, kv_heads, max_new, width, rc):
    """A sequence's units are counted in 32 bits; pages may be shared, so its memory does not bound them."""
    n = C.c_uint64(7)
    c = _lib.Kv4Cache(256, 256, 256, 256, 1000, 32, kv_heads, 64, width, width, 3)
    a = _lib.Kv4AttentionDesc(None, None, 0, 1, q_heads, max_new, (1 << 31) - 1, 0, 0, 0.1)
    assert lib.rldx_kv4_attention_workspace_size(C.byref(c), C.byref(a), C.byref(n)) == rc
