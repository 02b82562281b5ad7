"""Products with 4-bit weights over the range of fp32 activations that they take.

Tolerance, max |y - ref| / max |ref| <= 4 sqrt(n + 8) 2^-23 with n = ceil(K / min(group, 64)): the products are exact, sums are fp32.
Running sums take a step for each group (or 64 inputs), n at most, one after another, and a step's own 32, 64 or 128 products are added in
8 blocks of 16 at most; each addition rounds, or on the matrix units cuts, its result to within 2^-23 of it.  Terms of random
sign keep partial sums at the size of the results, so the n + 8 errors in a chain add up like the root of their number; 4 is
four standard deviations.
Where terms may have any sign the same factor is taken of the sum of magnitudes, which no partial sum exceeds."""
import numpy as np
import pytest

from test_q4_gpu import dense, product, weights

pytestmark = pytest.mark.gpu


def tol(K, group):
    return 4 * (-(-K // min(group, 64)) + 8) ** 0.5 * 2.0 ** -23


@pytest.fixture(scope="module")
def ctx():
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    yield c
    c.close()


@pytest.mark.parametrize("M", [1, 2, 5, 30])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_the_range_of_activations(ctx, M, group):
    """Up to 2^116 no sum of a group leaves fp32: 128 products of up to 8 times that.  Down to 2^-110 the planes hold all 24
    bits; below it a value is cut to a multiple of bfloat16's smallest step, 2^-133."""
    import shainet_b200 as S
    rng = np.random.default_rng(M + group)
    K, N = 384, 70
    packed, scales = weights(rng, K, N, group)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, group)
    w = dense(packed, scales, K, group)
    for top in (116, 60, 0, -60, -109):
        x = (rng.choice([-1.0, 1.0], (M, K)) * rng.uniform(0.5, 1.0, (M, K)) * 2.0 ** top).astype(np.float32)
        got, ref = product(ctx, W, x, N), x.astype(np.float64) @ w.T
        assert np.isfinite(got).all()
        assert np.abs(got - ref).max() <= tol(K, group) * (np.abs(x).astype(np.float64) @ np.abs(w).T).max() + K * 2.0 ** -149, top
    for top in (-115, -124, -130):
        x = (rng.standard_normal((M, K)) * 2.0 ** top).astype(np.float32)
        got, ref = product(ctx, W, x, N), x.astype(np.float64) @ w.T
        # per input: what is cut off, and subnormal sums' own step
        assert np.abs(got - ref).max() <= (tol(K, group) * np.abs(x).astype(np.float64) @ np.abs(w).T + 2.0 ** -133 * np.abs(w).sum(1) + K * 2.0 ** -149).max(), top
    W.close()
