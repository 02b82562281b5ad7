"""Refusals of the page step that also writes decode lengths; they need no device (arguments are looked at before the context)."""
import pytest

A, B, C_, D = 4096, 8192, 12288, 16384   # aligned addresses that are never followed


@pytest.fixture(scope="module")
def lib():
    from shainet_b200 import build, _lib
    build.build()
    return _lib.load()


def _step(lib, **kw):
    a = dict(ctx=None, requests=4, lens=A, delta=A, table=A, width=8, page_rows=16, free=A, num_pages=100, count=A, lens_out=B,
             count_out=A, first=A, slots=A, tokens=64, decode_lens=C_, status=A, stream=None)
    a.update(kw)
    return lib.shainet_attn_paged_step_dev(*a.values())


@pytest.mark.parametrize("kw,code,word", [
    (dict(decode_lens=None), "E_INVALID", "decode_lens"), (dict(decode_lens=A), "E_INVALID", "decode_lens"),
    (dict(decode_lens=B), "E_INVALID", "decode_lens"), (dict(decode_lens=C_ + 2), "E_INVALID", "aligned"),
    (dict(requests=-1), "E_INVALID", "requests"), (dict(requests=8193), "E_UNSUPPORTED", "at most 8192"),
    (dict(tokens=-1), "E_INVALID", "max_tokens"), (dict(page_rows=0), "E_INVALID", "page_rows"),
    (dict(num_pages=0), "E_INVALID", "pool"), (dict(width=0), "E_INVALID", "table_width"), (dict(status=None), "E_INVALID", "null array"),
    (dict(), "E_INVALID", "null context"), (dict(lens_out=A), "E_INVALID", "null context"),
    (dict(requests=0, lens=None, delta=None, table=None, lens_out=None, decode_lens=None), "E_INVALID", "null context"),
], ids=lambda v: str(v))
def test_step_refusals(lib, kw, code, word):
    from shainet_b200 import _lib
    assert _step(lib, **kw) == getattr(_lib, code)
    assert word in lib.shainet_attn_last_error().decode()
