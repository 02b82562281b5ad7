"""What kernels report to the host: a bad page and a wait that gave up are kept apart, so that neither hides the other, in
whichever order they happen.  The waits run out because nothing sets their words; no access is bad."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from shainet_b200 import build
    build.build()


def bad_slot(S, c, t):
    """A copy of one row to a slot outside its pool."""
    t["paged"].scatter_dev(t["attn"], t["kp"].data_ptr(), t["vp"].data_ptr(), 2, t["slots"].data_ptr(), 0, 1)


def lost_wait(S, c, t):
    c.comm_wait(8, 16, 12345)


@pytest.mark.parametrize("first,then", [(bad_slot, lost_wait), (lost_wait, bad_slot)], ids=["page_wait", "wait_page"])
def test_a_bad_page_and_a_lost_wait_are_both_reported(lib, first, then):
    import torch
    import shainet_b200 as S
    from shainet_b200 import _lib
    c = S.AttnContext(0)
    c.comm_open([c.comm_create(64)], 0)
    c.comm_set_wait_limit_ms(20)
    t = dict(attn=S.LlamaAttention(c, 8, 2, 64), paged=S.PagedAttention(c, 8, 2, 64, 16),
             slots=torch.tensor([32], dtype=torch.int32, device="cuda"))
    t["attn"].cache.fill_normal(4, 1)
    t["kp"], t["vp"] = (torch.zeros(2, 2, 16, 64, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    first(S, c, t)
    then(S, c, t)
    with pytest.raises(S.ShainetAttnError) as e:
        c.sync()
    assert e.value.code == _lib.E_DEVICE_WAIT
    with pytest.raises(S.ShainetAttnError) as e:
        c.sync()
    assert e.value.code == _lib.E_INVALID and "outside" in str(e.value)
    c.sync()
    assert not t["kp"].any() and not t["vp"].any()
    # either by itself still is what it was
    for call, code in ((bad_slot, _lib.E_INVALID), (lost_wait, _lib.E_DEVICE_WAIT)):
        call(S, c, t)
        with pytest.raises(S.ShainetAttnError) as e:
            c.sync()
        assert e.value.code == code
        c.sync()
    t["paged"].close()
    t["attn"].close()
    c.close()
