"""Refusals of the paged and 4-bit entries that need no device (arguments are looked at before the context), and the index
arithmetic of pages, compiled here with the host compiler."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 4096   # an aligned address that is never followed


@pytest.fixture(scope="module")
def lib():
    from shainet_b200 import build, _lib
    build.build()
    return _lib.load()


def _plan(lib, **kw):
    a = dict(ctx=None, requests=4, lens=A, delta=A, table=A, width=8, page_rows=16, free=A, num_pages=100, count=A, lens_out=A,
             count_out=A, first=A, slots=A, tokens=64, status=A, stream=None)
    a.update(kw)
    return lib.shainet_attn_paged_plan_dev(*a.values())


@pytest.mark.parametrize("kw,code,word", [
    (dict(requests=-1), "E_INVALID", "requests"), (dict(requests=8193), "E_UNSUPPORTED", "at most 8192"),
    (dict(tokens=-1), "E_INVALID", "max_tokens"), (dict(page_rows=0), "E_INVALID", "page_rows"),
    (dict(page_rows=4097), "E_INVALID", "page_rows"), (dict(num_pages=0), "E_INVALID", "pool"),
    (dict(num_pages=1 << 27, page_rows=16), "E_INVALID", "2^31"), (dict(width=0), "E_INVALID", "table_width"),
    (dict(requests=4096, width=1 << 20), "E_INVALID", "cells"), (dict(lens=None), "E_INVALID", "null array"),
    (dict(status=None), "E_INVALID", "null array"), (dict(slots=None), "E_INVALID", "null array"),
    (dict(first=A + 2), "E_INVALID", "aligned"), (dict(), "E_INVALID", "null context"),
    (dict(slots=None, tokens=0), "E_INVALID", "null context"),
    (dict(requests=0, lens=None, delta=None, table=None, lens_out=None), "E_INVALID", "null context"),
], ids=lambda v: str(v))
def test_plan_refusals(lib, kw, code, word):
    from shainet_b200 import _lib
    assert _plan(lib, **kw) == getattr(_lib, code)
    assert word in lib.shainet_attn_last_error().decode()


@pytest.mark.parametrize("args,code,word", [
    ((8, 3, 64, 16, 0), "E_INVALID", "8 query heads over 3"), ((0, 1, 64, 16, 0), "E_INVALID", "query heads"),
    ((8, 2, 96, 16, 0), "E_UNSUPPORTED", "head_dim 96"), ((8, 2, 64, 0, 0), "E_INVALID", "page_rows"),
    ((8, 2, 64, 16, 2), "E_INVALID", "format"), ((8, 2, 64, 16, 1), "E_INVALID", "null context"),
], ids=lambda v: str(v))
def test_paged_create_refusals(lib, args, code, word):
    from shainet_b200 import _lib
    h = C.c_void_p(5)
    assert lib.shainet_attn_paged_create(None, C.byref(h), *args) == getattr(_lib, code)
    assert word in lib.shainet_attn_last_error().decode() and not h.value
    assert lib.shainet_attn_paged_create(None, None, *args) == _lib.E_INVALID


def test_paged_calls_refuse_null_and_negative(lib):
    from shainet_b200 import _lib
    dec = lib.shainet_attn_paged_decode_dev
    assert dec(None, None, None, A, A, 10, A, A, A, A, A, 4, A, -1, 0.1, None) == _lib.E_INVALID
    assert dec(None, None, None, A, A, 10, A, A, A, A, A, 0, A, 1, 0.1, None) == _lib.E_INVALID
    assert b"table_width" in lib.shainet_attn_last_error()
    assert dec(None, None, None, A, A, 10, A, A, A, A, A, 4, A, 1, 0.1, None) == _lib.E_INVALID
    assert b"null context" in lib.shainet_attn_last_error()
    assert lib.shainet_attn_paged_scatter_dev(None, None, None, A, A, 10, A, -1, 4, None) == _lib.E_INVALID
    assert lib.shainet_attn_paged_scatter_dev(None, None, None, A, A, 10, A, 0, 4, None) == _lib.E_INVALID
    assert lib.shainet_attn_paged_gather_dev(None, None, None, A, A, 10, A, -4, None) == _lib.E_INVALID
    assert lib.shainet_attn_paged_destroy(None) == _lib.OK


def test_q4_refusals(lib):
    from shainet_b200 import _lib
    h = C.c_void_p(5)
    w = (C.c_float * 64)()
    assert lib.shainet_attn_q4_create(None, C.byref(h), w, 8, 8, 48) == _lib.E_UNSUPPORTED
    assert b"group 48" in lib.shainet_attn_last_error() and not h.value
    assert lib.shainet_attn_q4_create(None, C.byref(h), w, 0, 8, 32) == _lib.E_INVALID
    assert lib.shainet_attn_q4_create(None, C.byref(h), w, 8, 8, 32) == _lib.E_INVALID
    assert b"null context" in lib.shainet_attn_last_error()
    assert lib.shainet_attn_q4_create_raw(None, C.byref(h), None, w, 8, 8, 32) == _lib.E_INVALID
    assert lib.shainet_attn_q4_create_dev(None, C.byref(h), A, None, 8, 8, 32) == _lib.E_INVALID
    assert lib.shainet_attn_q4_gemv_dev(None, None, A, A, -1, None) == _lib.E_INVALID
    assert b"rows" in lib.shainet_attn_last_error()
    assert lib.shainet_attn_q4_gemv_dev(None, None, A, A, 1, None) == _lib.E_INVALID
    assert lib.shainet_attn_q4_export(None, A, w) == _lib.E_INVALID
    assert lib.shainet_attn_q4_destroy(None) == _lib.OK


def test_quantised_arrays_are_checked_before_the_library():
    import numpy as np
    import shainet_b200 as S

    class Ctx:
        L = h = None
    with pytest.raises(ValueError):
        S.Q4Weight.from_quantized(Ctx(), np.zeros((4, 8), np.uint8), np.zeros((4, 1), np.float32), 17, 32)
    with pytest.raises(ValueError):
        S.Q4Weight.from_quantized(Ctx(), np.zeros((4, 8), np.uint8), np.zeros((4, 2), np.float32), 16, 32)
    with pytest.raises(ValueError):
        S.PagedAttention(Ctx(), 8, 2, 64, 16, "f16")


_HOST = r"""
#include "paged_index.h"
using namespace shainet;
extern "C" {
int t_pages(int n, int p) { return pages_of(n, fast_div(p), p); }
int t_page(int page, int n) { return page_in_pool(page, n); }
int t_slot(int slot, int n, int p) { return slot_in_pool(slot, n, p); }
int t_len(int len, int w, int p) { return valid_len(len, max_len_of(w, p)); }
int t_div(int n, int d) { return divide(n, fast_div(d)); }
long long t_div_sweep(int d) {      // first n whose quotient is wrong, or -1: around every multiple up to 2^31 - 1, or a grid of them
    const FastDiv f = fast_div(d);
    const long long step = (2147483647ll / d / 20000 + 1) * d;
    for (long long m = 0; m <= 2147483647ll; m += step)
        for (long long n = m - 2; n <= m + 2; ++n)
            if (n >= 0 && n <= 2147483647ll && divide((int)n, f) != (int)(n / d)) return n;
    return divide(2147483647, f) == 2147483647 / d ? -1 : 2147483647;
}
unsigned long long t_row(int page, int kv, int h, int p, int r) { return pool_row(page, kv, h, p, r); }
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_index_arithmetic_keeps_bad_pages_out_and_64_bits(tmp_path):
    """What stands between a bad table cell, slot or length and an access: tested on the host before any GPU run."""
    src, so = tmp_path / "t.cpp", tmp_path / "t.so"
    src.write_text(_HOST)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "shainet_b200", "csrc"), str(src), "-o",
                    str(so)], check=True)
    L = C.CDLL(str(so))
    L.t_row.restype = C.c_ulonglong
    L.t_div_sweep.restype = C.c_longlong
    assert all(L.t_div_sweep(d) == -1 for d in [*range(1, 130), *range(131, 4097, 61), 4095, 4096])
    big = 2**31 - 1
    assert [L.t_pages(n, 16) for n in (0, 1, 16, 17)] == [0, 1, 1, 2] and L.t_pages(big, 1) == big and L.t_pages(big, 4096) == 1 << 19
    assert [L.t_page(p, 5) for p in (-1, 0, 4, 5, big, -big)] == [0, 1, 1, 0, 0, 0]
    assert [L.t_slot(s, 5, 16) for s in (-1, 0, 79, 80, big)] == [0, 1, 1, 0, 0]
    assert L.t_slot(big, 1 << 20, 4096) == 1          # the product is taken in 64 bits
    assert [L.t_len(n, 3, 16) for n in (-1, 0, 48, 49, big)] == [0, 0, 48, 0, 0] and L.t_len(big, 1 << 20, 4096) == big
    assert L.t_row(big - 1, 128, 127, 4096, 4095) == ((big - 1) * 128 + 127) * 4096 + 4095
