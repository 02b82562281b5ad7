"""Page plans at the last page: a step that takes every page there is, one that is a page short, one that frees as many as it
takes, with and without free pages, in one CTA and in the cluster (a longer array of slots), in place and not."""
import numpy as np
import pytest

from test_paged_plan_gpu import OK, SHORT, check, state

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    yield c
    c.close()


@pytest.mark.parametrize("in_place", [False, True], ids=["out", "in_place"])
@pytest.mark.parametrize("tokens", [249, 5000], ids=["one_cta", "cluster"])
@pytest.mark.parametrize("spare", [0, 1, 9])
def test_the_last_page(ctx, spare, tokens, in_place):
    """Requests 0, 2 and 5 free 3 + 2 + 1 pages of 16 rows, requests 3 and 4 take one each: request 1 may grow by 4 + spare."""
    rng = np.random.default_rng(5)
    P, W, room = 16, 24, 4 + spare
    lens = np.array([40, 0, 33, 48, 17, 60, 5], np.int32)
    table, free = state(rng, len(lens), W, P, 40, lens, spare)
    for grown, want, left in ((room * P, [OK, 0], 0), (room * P - 15, [OK, 0], 0), (room * P - 16, [OK, 0], 1),
                              (room * P + 1, [SHORT, 1], spare)):
        delta = np.array([-40, grown, -17, 1, 31, -21, 0], np.int32)
        got = check(ctx, lens, delta, table, P, free, spare, tokens, in_place=in_place)
        assert got[0] == want and got[2] == left, grown


@pytest.mark.parametrize("tokens", [40, 5000], ids=["one_cta", "cluster"])
def test_every_page_changes_hands(ctx, tokens):
    """A full pool: what one request gives up is exactly what another takes, then one row more."""
    rng = np.random.default_rng(6)
    P, W = 4, 10
    lens = np.array([40, 0, 3], np.int32)
    table, free = state(rng, 3, W, P, 11, lens, 0)
    assert check(ctx, lens, np.array([-36, 36, 1], np.int32), table, P, free, 0, tokens)[0] == [OK, 0]
    assert check(ctx, lens, np.array([-36, 36, 2], np.int32), table, P, free, 0, tokens)[0] == [SHORT, 1]
    assert check(ctx, lens, np.array([-35, 36, 1], np.int32), table, P, free, 0, tokens)[0] == [SHORT, 1]
