"""Refusals of the 4-bit entries that a kernel would otherwise meet as a misaligned address; they need no device."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from shainet_b200 import build, _lib
    build.build()
    return _lib.load()


@pytest.mark.parametrize("off,word", [(1, "4-byte aligned"), (2, "4-byte aligned"), (3, "4-byte aligned"), (0, "null context"), (4, "null context")])
def test_device_scales_are_aligned(lib, off, word):
    from shainet_b200 import _lib
    h = C.c_void_p(5)
    assert lib.shainet_attn_q4_create_dev(None, C.byref(h), 4096 + 1, 8192 + off, 8, 8, 32) == _lib.E_INVALID
    assert word in lib.shainet_attn_last_error().decode() and not h.value
