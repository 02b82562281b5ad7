"""Weights that the 4-bit quantiser can only just represent, and those that it cannot."""
import numpy as np
import pytest

from test_q4_gpu import dense

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    yield c
    c.close()


@pytest.mark.parametrize("size", [2.0 ** -120, 2.0 ** -126, 2.0 ** -130, 2.0 ** -140, 2.0 ** -148, 2.0 ** 127])
def test_quantiser_of_tiny_and_huge_groups(ctx, size):
    """A group whose 1 / scale is not finite: its zeros are zeros, and no value is further off than half a step of the scale and the
    roundings of values and scale to fp32's smallest step."""
    import shainet_b200 as S
    rng = np.random.default_rng(9)
    K, N = 96, 24
    w = (rng.uniform(-1.0, 1.0, (K, N)) * size).astype(np.float32)
    w[::5] = 0.0
    w[0, 0] = size
    W = S.Q4Weight.from_simple(ctx, w, 32)
    packed, scales = W.export()
    assert np.isfinite(scales).all() and (scales > 0).all()
    got = dense(packed, scales, K, 32).T
    assert (got[::5][w[::5] == 0] == 0).all()
    assert np.abs(got - w).max() <= (0.5 + 3 * 7.5 * 2.0 ** -24) * scales.max() + 8 * 2.0 ** -149
    W.close()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_weights_that_are_not_finite_are_refused(ctx, bad):
    import shainet_b200 as S
    from shainet_b200 import _lib
    w = np.ones((70, 5), np.float32)
    w[69, 4] = bad
    with pytest.raises(S.ShainetAttnError) as e:
        S.Q4Weight.from_simple(ctx, w, 64)
    assert e.value.code == _lib.E_INVALID and "not finite" in str(e.value)
