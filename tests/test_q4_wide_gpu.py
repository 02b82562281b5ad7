"""Products of one and two rows with 4-bit weights whose widths leave no room for the rows beside the weights.

Tolerance, max |y - ref| / max |ref| <= 4 sqrt(n + 8) 2^-23 with n = ceil(K / min(group, 64)): the products are exact, sums are fp32.
Running sums take a step for each group (or 64 inputs), n at most, one after another, and a step's own 32, 64 or 128 products are added in
8 blocks of 16 at most; each addition rounds, or on the matrix units cuts, its result to within 2^-23 of it.  Terms of random
sign keep partial sums at the size of the results, so the n + 8 errors in a chain add up like the root of their number; 4 is
four standard deviations."""
import numpy as np
import pytest

from helpers import rel_err
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


# one row's planes fit beside the rings up to 28992 inputs, two rows' up to 14464
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", [(1, 28672, 700), (1, 28992, 40), (1, 28993, 40), (1, 29056, 300), (1, 40001, 33), (2, 14464, 40), (2, 14465, 40),
                                   (2, 14528, 1000), (2, 28672, 4100), (3, 28672, 600), (2, 50000, 17), (1, 65536, 16)], ids=lambda v: str(v))
def test_wide_rows(ctx, M, K, N, group):
    import torch
    import shainet_b200 as S
    rng = np.random.default_rng(K + M + group)
    packed, scales = weights(rng, K, N, group)
    x = rng.standard_normal((M, K)).astype(np.float32)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, group)
    got = product(ctx, W, x, N)
    ref = x.astype(np.float64) @ dense(packed, scales, K, group).T
    assert rel_err(got, ref) <= tol(K, group), rel_err(got, ref)
    assert np.array_equal(got, product(ctx, W, x, N))
    W.close()


@pytest.mark.parametrize("M", [1, 2, 8, 40, 100])
def test_one_or_two_wide_rows_as_one_of_many(ctx, M):
    """Every row by itself, by twos and among the others agrees to both sides' tolerance."""
    import shainet_b200 as S
    rng = np.random.default_rng(M)
    K, N = 30000, 90
    packed, scales = weights(rng, K, N, 128)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, 128)
    x = rng.standard_normal((M, K)).astype(np.float32)
    got = product(ctx, W, x, N)
    for m in range(0, M, max(1, M // 4)):
        assert rel_err(got[m:m + 2], product(ctx, W, np.ascontiguousarray(x[m:m + 2]), N)) <= 2 * tol(K, 128)
    W.close()
