"""Products with 4-bit weights and group scales (shainet_attn_q4_*) against numpy in 64 bits.

Tolerance, max |y - ref| / max |ref| <= 2e-6 * max(1, sqrt(K / 4096)): an output is a sum of K exact products of 4-bit
values and fp32 activations, added in fp32.  Every addition rounds (or, on the matrix units, cuts) to within 2^-23 of a
partial sum; partial sums of independent terms are at most about the size of the result's scale, sqrt(K) terms, and a lane adds no more
than K / 4 of them before the rest is joined pairwise, so the errors add up like sqrt(K / 4) * 2^-23 * 0.5, 2e-6 at K = 4096."""
import numpy as np
import pytest

from helpers import rel_err

pytestmark = pytest.mark.gpu


def tol(K):
    return 2e-6 * max(1.0, (K / 4096) ** 0.5)


@pytest.fixture(scope="module")
def ctx():
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    yield c
    c.close()


def weights(rng, K, N, group):
    packed = rng.integers(0, 256, (N, (K + 1) // 2)).astype(np.uint8)
    scales = (0.004 * (0.6 + 0.8 * rng.random((N, -(-K // group))))).astype(np.float32)
    return packed, scales


def dense(packed, scales, K, group):
    q = np.stack([packed & 15, packed >> 4], -1).reshape(len(packed), -1)[:, :K].astype(np.float64) - 8
    return q * scales.astype(np.float64).repeat(group, 1)[:, :K]


def product(ctx, W, x, N, stream=None):
    import torch
    tx = torch.from_numpy(x).cuda()
    ty = torch.full((len(x) + 1, N), float("nan"), device="cuda")
    torch.cuda.synchronize()
    W.gemv_dev(tx.data_ptr(), ty.data_ptr(), len(x), stream=stream)
    torch.cuda.synchronize()
    ctx.sync()
    got = ty.cpu().numpy()
    assert np.isnan(got[len(x)]).all()
    return got[:len(x)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 130])
@pytest.mark.parametrize("K,N", [(2048, 512), (1000, 333)], ids=lambda v: str(v))
def test_rows(ctx, K, N, M, group):
    import shainet_b200 as S
    rng = np.random.default_rng(K + N + M + group)
    packed, scales = weights(rng, K, N, group)
    x = rng.standard_normal((M, K)).astype(np.float32)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, group)
    got = product(ctx, W, x, N)
    ref = x.astype(np.float64) @ dense(packed, scales, K, group).T
    assert rel_err(got, ref) <= tol(K), rel_err(got, ref)
    W.close()


# many tiles a CTA, blocks of inputs that end a group early, shared inputs of one to eight CTAs, one or more passes
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K,N,M", [(200, 40001, 33), (64, 80000, 25), (449, 39000, 64), (2052, 38000, 12), (192, 257, 40), (320, 513, 64), (5000, 100, 64),
                                   (4100, 4100, 24), (4097, 3900, 41), (12290, 300, 3), (9000, 5000, 8), (1000, 40, 1000), (1100, 900, 257)],
                         ids=lambda v: str(v))
def test_many_rows(ctx, K, N, M, group):
    import torch
    import shainet_b200 as S
    rng = np.random.default_rng(K + N + M + group)
    packed, scales = weights(rng, K, N, group)
    x = rng.standard_normal((M, K)).astype(np.float32)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, group)
    got = product(ctx, W, x, N)
    ref = (torch.from_numpy(x).cuda().double() @ torch.from_numpy(dense(packed, scales, K, group)).cuda().T).cpu().numpy()
    assert rel_err(got, ref) <= tol(K), rel_err(got, ref)
    assert np.array_equal(got, product(ctx, W, x, N))
    W.close()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K,N", [(1, 1), (2, 3), (31, 17), (32, 16), (33, 15), (63, 8), (65, 1), (127, 40), (129, 2), (255, 31), (513, 7), (2047, 100),
                                 (4097, 65), (12289, 24), (64, 20011)], ids=lambda v: str(v))
def test_odd_sizes(ctx, K, N, group):
    import shainet_b200 as S
    rng = np.random.default_rng(K * 3 + N + group)
    packed, scales = weights(rng, K, N, group)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, group)
    w = dense(packed, scales, K, group)
    for M in (1, 3, 11):
        x = rng.standard_normal((M, K)).astype(np.float32)
        got, ref = product(ctx, W, x, N), x.astype(np.float64) @ w.T
        # few terms may cancel: against the sum of magnitudes
        assert np.abs(got - ref).max() <= tol(K) * (np.abs(x).astype(np.float64) @ np.abs(w).T).max(), (M, rel_err(got, ref))
    W.close()


def test_every_nibble_and_exact_products(ctx):
    """x of few bits and scales that are powers of two: every sum is exact in fp32, so results have to be equal."""
    import shainet_b200 as S
    rng = np.random.default_rng(1)
    K, N = 256, 48
    packed, _ = weights(rng, K, N, 32)
    assert len(np.unique(packed)) == 256
    scales = np.float32(2.0) ** rng.integers(-3, 4, (N, K // 32)).astype(np.float32)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, 32)
    for M in (1, 2, 7, 40):
        x = rng.integers(-8, 9, (M, K)).astype(np.float32)
        assert np.array_equal(product(ctx, W, x, N), (x.astype(np.float64) @ dense(packed, scales, K, 32).T).astype(np.float32))
    # each row of the identity picks one column of the weight: exact to the scale's rounding
    eye = np.eye(K, dtype=np.float32)
    scales = (0.004 * (0.6 + 0.8 * rng.random((N, K // 32)))).astype(np.float32)
    V = S.Q4Weight.from_quantized(ctx, packed, scales, K, 32)
    assert np.array_equal(product(ctx, V, eye, N), dense(packed, scales, K, 32).T.astype(np.float32))
    W.close()
    V.close()


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e12, 1e30])
def test_small_and_large_activations(ctx, size):
    """All of fp32's range: x is not rounded to fewer bits, rows of very different size do not touch each other."""
    import shainet_b200 as S
    rng = np.random.default_rng(2)
    K, N = 512, 96
    packed, scales = weights(rng, K, N, 64)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, 64)
    w = dense(packed, scales, K, 64)
    x = rng.standard_normal((3, K)).astype(np.float32)
    x[1] *= np.float32(size)
    got, ref = product(ctx, W, x, N), x.astype(np.float64) @ w.T
    for m in range(3):
        assert rel_err(got[m], ref[m]) <= tol(K), (m, rel_err(got[m], ref[m]))
    W.close()


def test_infinite_and_nan_activations_stay_in_their_row(ctx):
    import shainet_b200 as S
    rng = np.random.default_rng(3)
    K, N = 300, 40
    packed, scales = weights(rng, K, N, 32)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, 32)
    for M in (2, 9, 20):
        x = rng.standard_normal((M, K)).astype(np.float32)
        clean = product(ctx, W, x, N)
        x[1, 7] = np.nan
        got = product(ctx, W, x, N)
        assert np.isnan(got[1]).all() and np.array_equal(np.delete(got, 1, 0), np.delete(clean, 1, 0))
        x[1, 7] = np.inf
        got = product(ctx, W, x, N)
        assert not np.isfinite(got[1]).any() and np.array_equal(np.delete(got, 1, 0), np.delete(clean, 1, 0))
    W.close()


@pytest.mark.parametrize("K,N,M", [(300, 40, 33), (300, 40, 64), (9000, 40, 3), (2000, 300, 10), (2000, 40000, 12)], ids=lambda v: str(v))
def test_rows_of_one_pass_do_not_touch_each_other(ctx, K, N, M):
    import shainet_b200 as S
    rng = np.random.default_rng(13)
    packed, scales = weights(rng, K, N, 64)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, 64)
    x = rng.standard_normal((M, K)).astype(np.float32)
    clean = product(ctx, W, x, N)
    for bad in (np.nan, np.inf, -np.inf, 3e38):
        x[1, K - 1] = bad
        got = product(ctx, W, x, N)
        assert np.array_equal(np.delete(got, 1, 0), np.delete(clean, 1, 0))
        if not np.isfinite(bad):
            assert not np.isfinite(got[1]).any()
    W.close()


@pytest.mark.parametrize("K,N,M", [(1, 1, 25), (31, 17, 64), (65, 15, 130), (12300, 1, 9), (127, 257, 33)], ids=lambda v: str(v))
def test_odd_sizes_of_many_rows(ctx, K, N, M):
    import shainet_b200 as S
    for group in (32, 64, 128):
        rng = np.random.default_rng(K + N + M + group)
        packed, scales = weights(rng, K, N, group)
        W = S.Q4Weight.from_quantized(ctx, packed, scales, K, group)
        w, x = dense(packed, scales, K, group), rng.standard_normal((M, K)).astype(np.float32)
        got, ref = product(ctx, W, x, N), x.astype(np.float64) @ w.T
        assert np.abs(got - ref).max() <= tol(K) * (np.abs(x).astype(np.float64) @ np.abs(w).T).max(), rel_err(got, ref)
        W.close()


def test_many_rows_on_two_streams_and_in_graphs(ctx):
    """Clusters and tensor memory under load: products of several shapes at once on two streams, then two graphs of them
    replayed at once; every result is bit for bit that of a call by itself."""
    import torch
    import shainet_b200 as S
    rng = np.random.default_rng(21)
    made = []
    for K, N, M, group in ((2048, 4100, 33, 128), (4096, 4096, 64, 64), (5000, 100, 40, 32), (2048, 20000, 12, 64)):
        packed, scales = weights(rng, K, N, group)
        W = S.Q4Weight.from_quantized(ctx, packed, scales, K, group)
        x = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).cuda()
        ys = [torch.full((M, N), float("nan"), device="cuda") for _ in range(3)]
        torch.cuda.synchronize()
        W.gemv_dev(x.data_ptr(), ys[0].data_ptr(), M)
        made.append((W, x, ys, M))
    ctx.sync()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(20):
        for i, s in enumerate(streams):
            for W, x, ys, M in made[:: 1 - 2 * i]:
                W.gemv_dev(x.data_ptr(), ys[1 + i].data_ptr(), M, stream=s.cuda_stream)
    torch.cuda.synchronize()
    ctx.sync()
    assert all(torch.equal(ys[0], y) for _, _, ys, _ in made for y in ys[1:])
    graphs = []
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for W, x, ys, M in made[:: 1 - 2 * i]:
                W.gemv_dev(x.data_ptr(), ys[1 + i].data_ptr(), M, stream=s.cuda_stream)
        graphs.append(g)
    for _, _, ys, _ in made:
        for y in ys[1:]:
            y.fill_(float("nan"))
    torch.cuda.synchronize()
    for rep in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    ctx.sync()
    assert all(torch.equal(ys[0], y) for _, _, ys, _ in made for y in ys[1:])
    for W, _, _, _ in made:
        W.close()


@pytest.mark.parametrize("K,N,group", [(2048, 512, 32), (1001, 77, 64), (130, 3, 128)], ids=lambda v: str(v))
def test_creation_and_export(ctx, K, N, group):
    """The three ways in hold the same weight; export gives back what went in; the quantiser follows its definition."""
    import torch
    import shainet_b200 as S
    rng = np.random.default_rng(K)
    w = (0.05 * rng.standard_normal((K, N))).astype(np.float32)
    w[:group, 0] = 0.0                                  # an all-zero group
    W = S.Q4Weight.from_simple(ctx, w, group)
    packed, scales = W.export()
    groups = -(-K // group)
    padded = np.zeros((groups * group, N), np.float32)
    padded[:K] = w
    amax = np.abs(padded.reshape(groups, group, N)).max(1).T                 # [N, groups]
    want_s = np.where(amax > 0, amax / np.float32(7.0), np.float32(1.0)).astype(np.float32)
    inv = (np.float32(1.0) / want_s).astype(np.float32)
    want_q = np.clip(np.rint((padded.T.reshape(N, groups, group) * inv[:, :, None]).astype(np.float32)), -7, 7).reshape(N, -1)[:, :K] + 8
    assert np.array_equal(scales, want_s)
    q = np.stack([packed & 15, packed >> 4], -1).reshape(N, -1)
    assert np.array_equal(q[:, :K], want_q)
    if K % 2:
        assert (packed[:, -1] >> 4 == 8).all()
    # half a step of the scale, and the roundings of inv, w * inv and q * s (three half steps of a value up to 7.5)
    assert np.abs(dense(packed, scales, K, group) - w.T).max() <= (0.5 + 3 * 7.5 * 2.0 ** -24) * scales.max()
    R = S.Q4Weight.from_quantized(ctx, packed, scales, K, group)
    tp, ts = torch.from_numpy(packed).cuda(), torch.from_numpy(scales).cuda()
    torch.cuda.synchronize()
    D = S.Q4Weight.from_device(ctx, tp.data_ptr(), ts.data_ptr(), K, N, group)
    tp.zero_(), ts.zero_()                              # nothing of the arrays is kept
    torch.cuda.synchronize()
    for X in (R, D):
        p2, s2 = X.export()
        assert np.array_equal(p2, packed) and np.array_equal(s2, scales)
    for M in (1, 12):
        x = rng.standard_normal((M, K)).astype(np.float32)
        ys = [product(ctx, X, x, N) for X in (W, R, D)]
        assert np.array_equal(ys[0], ys[1]) and np.array_equal(ys[0], ys[2])
    for X in (W, R, D):
        X.close()


def test_streams_graphs_and_repeats_are_bit_identical(ctx):
    import torch
    import shainet_b200 as S
    rng = np.random.default_rng(4)
    K, N = 2048, 1024
    packed, scales = weights(rng, K, N, 32)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, 32)
    for M in (1, 6, 33):
        tx = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).cuda()
        ys = [torch.full((M, N), float("nan"), device="cuda") for _ in range(4)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        W.gemv_dev(tx.data_ptr(), ys[0].data_ptr(), M)
        ctx.sync()
        for rep in range(10):                          # two calls at once
            for s, y in zip(streams, ys[1:3]):
                W.gemv_dev(tx.data_ptr(), y.data_ptr(), M, stream=s.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            W.gemv_dev(tx.data_ptr(), ys[3].data_ptr(), M, stream=streams[0].cuda_stream)
        ys[3].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(ys[0], y) for y in ys[1:])
    W.close()


def test_refusals_with_a_device(ctx):
    import torch
    import shainet_b200 as S
    from shainet_b200 import _lib
    rng = np.random.default_rng(5)
    packed, scales = weights(rng, 64, 16, 32)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, 64, 32)
    t = torch.zeros(1024, device="cuda")
    W.gemv_dev(t.data_ptr(), t.data_ptr(), 0)
    for args in ((t.data_ptr() + 4, t.data_ptr(), 1), (t.data_ptr(), t.data_ptr() + 8, 1), (None, t.data_ptr(), 1), (t.data_ptr(), t.data_ptr(), -1)):
        with pytest.raises(S.ShainetAttnError) as e:
            W.gemv_dev(*args)
        assert e.value.code == _lib.E_INVALID
    other = S.AttnContext(0)
    assert other.L.shainet_attn_q4_gemv_dev(other.h, W.h, t.data_ptr(), t.data_ptr() + 2048, 1, None) == _lib.E_INVALID
    other.close()
    W.close()
