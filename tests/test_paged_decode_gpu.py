"""Attention of one new token per request over pages (shainet_attn_paged_decode_dev) against numpy in 64 bits.

Tolerance of the outputs, max |y - ref| / max |ref| <= DECODE_TOL = 1e-5, the framework's class for fp32 decode: a score is a
sum of head_dim products of fp32 values with |score| up to about 6, whose roundings add up like sqrt(head_dim + 8) half
steps of 2^-24 of partial sums of that size, 12 * 6 * 6e-8 = 4e-6 at most in the exponent of a weight; a weighted mean over
rows has no more than its weights have, and the sums over rows are joined from partial sums of fp32, which adds less.
The rows written into the pages: fp32 rows within 4e-7 of the largest entry (three roundings and a sine of 2 ulp, as the
framework's own append tests allow), 16-bit rows within half a step, 2^-8 relative, plus that."""
import numpy as np
import pytest

from helpers import DECODE_TOL, L1B, Q30, Q8B, norm_weights, rel_err

pytestmark = pytest.mark.gpu
ROW_TOL = 4e-7
LAYOUTS = {"L1B": L1B, "Q8B": Q8B, "Q30": Q30, "mha": dict(H=16, KV=16, hd=64, theta=1e4), "g2": dict(H=4, KV=2, hd=128, theta=1e4),
           "g3": dict(H=6, KV=2, hd=128, theta=5e5), "g5": dict(H=10, KV=2, hd=64, theta=5e5),
           "g7": dict(H=28, KV=4, hd=128, theta=1e6, bias=True), "g12": dict(H=12, KV=1, hd=64, theta=1e6, bias=True, qk_norm=True),
           "g16": dict(H=32, KV=2, hd=128, theta=1e6), "g24": dict(H=24, KV=1, hd=128, theta=1e4, qk_norm=True),
           "g40": dict(H=40, KV=1, hd=64, theta=1e4), "one": dict(H=1, KV=1, hd=128, theta=1e4)}


@pytest.fixture(scope="module")
def ctx():
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    yield c
    c.close()


class Batch:
    """Pages with stale, infinite and NaN values wherever no request has a position, tables with distinct random pages and
    cells out of the pool behind them, raw projections, and the parameters of the block."""

    def __init__(self, ctx, layout, lens, P, kv, seed, spread=1.0, extra_width=2):
        import torch
        import shainet_b200 as S
        self.rng = rng = np.random.default_rng(seed)
        self.sh, self.P, self.kv, self.lens = layout, P, kv, np.asarray(lens, np.int32)
        H, KV, hd = layout["H"], layout["KV"], layout["hd"]
        B = len(lens)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)
        held = [-(-int(n) // P) for n in lens]
        self.W = max(max(held), 1) + extra_width
        self.NP = sum(held) + 2
        order = rng.permutation(self.NP).astype(np.int32)
        self.table = np.full((B, self.W), 2**31 - 1, np.int32)
        at = 0
        for b, n in enumerate(held):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.k, self.v = f(self.NP, KV, P, hd), f(self.NP, KV, P, hd)
        if kv == "bf16":
            self.k, self.v = (torch.from_numpy(x).bfloat16().float().numpy() for x in (self.k, self.v))
        live = np.zeros((self.NP, P), bool)
        for b, n in enumerate(lens):
            for p in range(max(0, int(n) - 1)):      # the new token's row is not there yet
                live[self.table[b, p // P], p % P] = True
        for x in (self.k, self.v):
            bad = np.array([np.nan, np.inf, -np.inf], np.float32)[rng.integers(0, 3, (self.NP, 1, P, hd))]
            x[:] = np.where(live[:, None, :, None], x, bad)
        self.live = live
        self.q, self.kn, self.vn = spread * f(B, H * hd), f(B, KV * hd), f(B, KV * hd)
        self.kw = {}
        if layout.get("qk_norm"):
            self.kw.update(q_norm=norm_weights(rng, hd), k_norm=norm_weights(rng, hd))
        if layout.get("bias"):
            self.kw.update(b_q=0.1 * f(H * hd), b_k=0.1 * f(KV * hd), b_v=0.1 * f(KV * hd))
        self.attn = S.LlamaAttention(ctx, H, KV, hd, layout["theta"], 1e-6, kv_format=kv, **self.kw)
        self.paged = S.PagedAttention(ctx, H, KV, hd, P, kv)
        self.ctx, self.scale = ctx, float(np.float32(1 / np.sqrt(hd)))
        dt = torch.float32 if kv == "f32" else torch.bfloat16
        dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
        self.tk, self.tv = dev(self.k).to(dt), dev(self.v).to(dt)
        self.tq, self.tkn, self.tvn, self.tt, self.tl = dev(self.q), dev(self.kn), dev(self.vn), dev(self.table), dev(self.lens)
        self.out = torch.full((B + 1, H * hd), float("nan"), device="cuda")
        torch.cuda.synchronize()

    def call(self, stream=None, requests=None, paged=None, num_pages=None):
        (paged or self.paged).decode_dev(self.attn, self.tk.data_ptr(), self.tv.data_ptr(), num_pages or self.NP, self.tq.data_ptr(),
                                         self.tkn.data_ptr(), self.tvn.data_ptr(), self.out.data_ptr(), self.tt.data_ptr(), self.W,
                                         self.tl.data_ptr(), len(self.lens) if requests is None else requests, self.scale, stream=stream)

    def run(self):
        import torch
        self.call()
        self.ctx.sync()
        torch.cuda.synchronize()
        got = self.out.cpu().numpy()
        assert np.isnan(got[len(self.lens):]).all()
        return got[:len(self.lens)], self.tk.float().cpu().numpy(), self.tv.float().cpu().numpy()

    def new_rows(self, b):
        """(q [H, hd], k [KV, hd], v [KV, hd]) of request b in 64 bits."""
        sh, hd = self.sh, self.sh["hd"]
        inv = np.array([np.float32(1.0 / sh["theta"] ** (2.0 * i / hd)) for i in range(hd // 2)], np.float32)
        ang = (np.float32(self.lens[b] - 1) * inv).astype(np.float32).astype(np.float64)
        c, s = np.cos(ang), np.sin(ang)
        res = []
        for x, heads, bias, norm in ((self.q, sh["H"], "b_q", "q_norm"), (self.kn, sh["KV"], "b_k", "k_norm"), (self.vn, sh["KV"], "b_v", None)):
            x = x[b].astype(np.float64) + self.kw.get(bias, np.zeros(1)).astype(np.float64)
            x = x.reshape(heads, hd)
            if norm in self.kw:
                x = x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-6) * self.kw[norm].astype(np.float64)
            if bias != "b_v":
                a, d = x[:, :hd // 2], x[:, hd // 2:]
                x = np.concatenate([a * c - d * s, d * c + a * s], 1)
            res.append(x)
        return res

    def check(self, tol=DECODE_TOL):
        got, gk, gv = self.run()
        sh, P, hd = self.sh, self.P, self.sh["hd"]
        G = sh["H"] // sh["KV"]
        want_k, want_v = self.k.copy(), self.v.copy()
        for b, n in enumerate(self.lens):
            if n == 0:
                assert (got[b] == 0).all()
                continue
            q, k, v = self.new_rows(b)
            page, row = self.table[b, (n - 1) // P], (n - 1) % P
            for pages, want, new in ((gk, want_k, k), (gv, want_v, v)):
                stored = pages[page, :, row]
                step = 0.0 if self.kv == "f32" else 2.0 ** -8
                assert (np.abs(stored - new) <= step * np.abs(new) + ROW_TOL * np.abs(new).max()).all()
                want[page, :, row] = stored         # attention sees the row as it is stored
            pos = np.arange(n)
            K = want_k[self.table[b, pos // P], :, pos % P].astype(np.float64)      # [n, KV, hd]
            V = want_v[self.table[b, pos // P], :, pos % P].astype(np.float64)
            s = np.einsum("kgd,nkd->kgn", q.reshape(sh["KV"], G, hd), K) * self.scale
            p = np.exp(s - s.max(-1, keepdims=True))
            ref = np.einsum("kgn,nkd->kgd", p / p.sum(-1, keepdims=True), V).reshape(-1)
            assert np.isfinite(got[b]).all(), b
            assert rel_err(got[b], ref) <= tol, (b, int(n), rel_err(got[b], ref))
        # nothing but the new rows was written (bit for bit: NaN rows stay what they were)
        assert np.array_equal(gk, want_k, equal_nan=True) and np.array_equal(gv, want_v, equal_nan=True)
        return got

    def close(self):
        self.paged.close()
        self.attn.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_ragged_batch_of_every_layout(ctx, layout, kv):
    """Lengths 0, 1, around tiles and pages, and a long one, in one batch; padded rows first, in the middle and last."""
    b = Batch(ctx, LAYOUTS[layout], [0, 1, 2, 15, 16, 17, 0, 31, 33, 64, 65, 130, 700, 1, 0], 16, kv, 100 + len(layout))
    b.check()
    b.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("P", [1, 2, 3, 7, 8, 24, 100, 256, 4096])
def test_page_sizes(ctx, P, kv):
    for layout, seed in (("L1B", 1), ("Q30", 2)):
        b = Batch(ctx, LAYOUTS[layout], [5, 100, 257, 1, 1023], P, kv, 31 * P + seed)
        b.check()
        b.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("layout,lens", [("L1B", [1]), ("L1B", [4097]), ("Q8B", [20011]), ("g16", [9001]), ("mha", [6000]), ("Q30", [33000, 3]),
                                         ("g7", [1] * 40 + [5000]), ("one", [30000]), ("L1B", list(range(1, 200)))], ids=lambda v: str(v)[:20])
def test_splits_of_few_and_many(ctx, layout, lens, kv):
    """One long request over the whole device, long beside short, many short ones."""
    b = Batch(ctx, LAYOUTS[layout], lens, 16, kv, len(lens) + 7)
    b.check()
    b.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_peaked_and_far_scores(ctx, kv):
    """Scores of some hundreds: a maximum that comes late, in another split, and takes all the weight.  A score's rounding is
    sqrt(136) half steps of 2^-24 of its size, here 400: 12 * 400 * 6e-8 = 2.9e-4 in the exponent of a weight that is not
    the largest; such weights' errors are held by the largest weight's share."""
    b = Batch(ctx, LAYOUTS["Q8B"] | dict(qk_norm=False), [3000, 40, 900], 16, kv, 77, spread=40.0)
    b.check(tol=3e-4)
    b.close()


def test_same_call_twice_and_on_another_stream_is_bit_identical(ctx):
    import torch
    b = Batch(ctx, LAYOUTS["Q8B"], [5000, 1, 0, 777, 12000], 16, "bf16", 9)
    first = b.run()
    side = torch.cuda.Stream()
    for stream in (None, side.cuda_stream, 0):
        b.out.fill_(float("nan"))
        torch.cuda.synchronize()
        b.call(stream=stream)
        torch.cuda.synchronize()
        ctx.sync()
        assert np.array_equal(first[0], b.out.cpu().numpy()[:5])
    b.close()


def test_two_handles_on_two_streams_at_once(ctx):
    import torch
    import shainet_b200 as S
    bs = [Batch(ctx, LAYOUTS["L1B"], [9000 + 100 * i, 30], 16, "f32", 50 + i) for i in range(2)]
    want = [b.run()[0] for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    for rep in range(20):
        for b, s in zip(bs, streams):
            b.call(stream=s.cuda_stream)
    torch.cuda.synchronize()
    ctx.sync()
    for b, w in zip(bs, want):
        assert np.array_equal(w, b.out.cpu().numpy()[:2])
        b.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_replayed_graph_follows_growing_requests(ctx, kv):
    """One capture; lengths, tables and pages change on the device between replays, from nothing to several splits."""
    import torch
    b = Batch(ctx, LAYOUTS["g7"] | dict(bias=False), [1, 40, 0, 3000], 16, kv, 21)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        b.call(stream=stream.cuda_stream)
    for lens in ([1, 33, 0, 5], [0, 0, 0, 0], [7, 40, 0, 2999], [1, 1, 1, 1]):
        c = Batch(ctx, LAYOUTS["g7"] | dict(bias=False), lens, 16, kv, 23 + sum(lens))      # the same parameters, other contents
        b.tk[:c.NP].copy_(c.tk), b.tv[:c.NP].copy_(c.tv)
        want = c.check()
        b.tl.copy_(c.tl), b.tq.copy_(c.tq), b.tkn.copy_(c.tkn), b.tvn.copy_(c.tvn)
        b.tt.fill_(2**31 - 1)
        b.tt[:, :c.W].copy_(c.tt)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ctx.sync()
        assert np.array_equal(b.out.cpu().numpy()[:4], want)
        assert torch.equal(b.tk[:c.NP].view(torch.uint8), c.tk.view(torch.uint8)) and torch.equal(b.tv[:c.NP].view(torch.uint8), c.tv.view(torch.uint8))
        c.close()
    b.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_pages_that_are_only_read_may_be_shared(ctx, kv):
    """Three requests with one prefix: their tables name the same pages up to the one that each writes into."""
    import torch
    b = Batch(ctx, LAYOUTS["L1B"], [100, 75, 70], 16, kv, 61)
    b.table[1, :4] = b.table[2, :4] = b.table[0, :4]
    b.tt.copy_(torch.from_numpy(b.table))
    torch.cuda.synchronize()
    b.check()
    b.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.125], ids=["zero", "negative"])
def test_other_scales(ctx, scale, kv):
    b = Batch(ctx, LAYOUTS["L1B"], [1, 33, 500], 16, kv, 62)
    b.scale = scale
    b.check()
    b.close()


def test_a_thousand_short_requests(ctx):
    rng = np.random.default_rng(63)
    b = Batch(ctx, LAYOUTS["one"], rng.integers(0, 40, 1000), 8, "f32", 64)
    b.check()
    b.close()


def test_no_request_and_layout_refusals(ctx):
    import shainet_b200 as S
    from shainet_b200 import _lib
    b = Batch(ctx, LAYOUTS["L1B"], [3, 4], 16, "f32", 3)
    b.call(requests=0)
    ctx.sync()
    assert np.isnan(b.out.cpu().numpy()).all()
    other = S.PagedAttention(ctx, 32, 8, 64, 16, "bf16")
    for paged in (other,):
        with pytest.raises(S.ShainetAttnError) as e:
            b.call(paged=paged)
        assert e.value.code == _lib.E_INVALID and "layout or format" in str(e.value)
    ctx2 = S.AttnContext(0)
    foreign = S.PagedAttention(ctx2, 32, 8, 64, 16, "f32")
    with pytest.raises(S.ShainetAttnError) as e:
        b.call(paged=foreign)
    assert "another context" in str(e.value)
    with pytest.raises(S.ShainetAttnError) as e:
        ctx2.close()
    assert e.value.code == _lib.E_STATE
    foreign.close()
    ctx2.close()
    b.tq = b.tq.flatten()[1:]
    with pytest.raises(S.ShainetAttnError) as e:
        b.call()
    assert "16-byte" in str(e.value)
    other.close()
    b.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_bad_pages_and_lengths_are_reported_and_not_followed(ctx, kv):
    """Table cells outside the pool and lengths outside the table: no access, an error at the next blocking call, the
    other requests unharmed."""
    import shainet_b200 as S
    from shainet_b200 import _lib
    for what in ("page", "negative_page", "new_page", "length", "negative_length"):
        b = Batch(ctx, LAYOUTS["L1B"], [100, 200, 300], 16, kv, 4)
        good = b.run()[0]
        if what == "page": b.tt[1, 3] = b.NP
        if what == "negative_page": b.tt[1, 3] = -1
        if what == "new_page": b.tt[1, 12] = 2**31 - 1
        if what == "length": b.tl[1] = b.W * 16 + 1
        if what == "negative_length": b.tl[1] = -5
        b.call()
        with pytest.raises(S.ShainetAttnError) as e:
            ctx.sync()
        assert e.value.code == _lib.E_INVALID and "outside" in str(e.value)
        ctx.sync()
        got = b.out.cpu().numpy()
        assert rel_err(got[0], good[0]) <= DECODE_TOL and rel_err(got[2], good[2]) <= DECODE_TOL
        if "length" in what:
            assert (got[1] == 0).all()
        b.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_offsets_past_32_bits(ctx, kv):
    """A pool of more than 2^32 bytes per tensor (2^31 elements at 16 bits): the request's pages are its last ones."""
    import torch
    import shainet_b200 as S
    H, KV, hd, P, n = 4, 2, 128, 1024, 700
    es = 4 if kv == "f32" else 2
    NP = (1 << 32) // (KV * P * hd * 2) + 3      # more than 2^31 elements at either size
    free = torch.cuda.mem_get_info()[0]
    if free < 2 * NP * KV * P * hd * es + (8 << 30):
        pytest.skip("not enough free device memory")
    dt = torch.float32 if kv == "f32" else torch.bfloat16
    kp, vp = (torch.empty(NP, KV, P, hd, dtype=dt, device="cuda") for _ in range(2))
    assert kp.numel() > 2**31
    sh = dict(H=H, KV=KV, hd=hd, theta=1e4)
    small = Batch(ctx, sh, [n], P, kv, 88)
    want = small.check()
    at = NP - 1
    kp[at].copy_(small.tk[small.table[0, 0]]), vp[at].copy_(small.tv[small.table[0, 0]])
    small.tk, small.tv, small.NP = kp, vp, NP
    small.tt[0, 0] = at
    small.out.fill_(float("nan"))
    torch.cuda.synchronize()
    small.call()
    ctx.sync()
    assert np.array_equal(small.out.cpu().numpy()[:1], want)
    small.close()


# ---- copies between pages and a contiguous cache ----

@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("layout,P,n,row0,rows", [("L1B", 16, 100, 0, 100), ("Q8B", 24, 777, 300, 477), ("Q30", 1, 5, 4, 1), ("mha", 256, 2000, 0, 1999),
                                                  ("one", 7, 33, 32, 1), ("g12", 16, 40, 0, 0)])
def test_scatter_and_gather(ctx, layout, P, n, row0, rows, kv):
    import torch
    import shainet_b200 as S
    rng = np.random.default_rng(n + P)
    sh = LAYOUTS[layout]
    H, KV, hd = sh["H"], sh["KV"], sh["hd"]
    attn = S.LlamaAttention(ctx, H, KV, hd, kv_format=kv)
    paged = S.PagedAttention(ctx, H, KV, hd, P, kv)
    dt = torch.float32 if kv == "f32" else torch.bfloat16
    k, v = (torch.from_numpy(rng.standard_normal((KV, n, hd)).astype(np.float32)).to(dt).float().numpy() for _ in range(2))
    attn.cache.import_(k, v)
    NP = -(-n // P) + 3
    table = torch.from_numpy(rng.permutation(NP).astype(np.int32)).cuda()
    pos = np.arange(row0, row0 + rows)
    slots = (table.cpu().numpy()[pos // P] * P + pos % P).astype(np.int32)
    skipped = rng.random(rows) < 0.1
    ts = torch.from_numpy(np.where(skipped, -1 - slots, slots).astype(np.int32)).cuda()
    kp, vp = (torch.full((NP, KV, P, hd), float("nan"), dtype=dt, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    paged.scatter_dev(attn, kp.data_ptr(), vp.data_ptr(), NP, ts.data_ptr(), row0, rows)
    ctx.sync()
    for pages, rows_of in ((kp, k), (vp, v)):
        want = np.full((NP, KV, P, hd), np.nan, np.float32)
        for i, s in enumerate(slots):
            if not skipped[i]:
                want[s // P, :, s % P] = rows_of[:, row0 + i]
        assert np.array_equal(pages.float().cpu().numpy(), want, equal_nan=True)
    # back: pages with finite rows, into a cache of another length
    for x in (kp, vp):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(dt))
    attn.cache.truncate(min(1, n))
    torch.cuda.synchronize()
    paged.gather_dev(attn, kp.data_ptr(), vp.data_ptr(), NP, table.data_ptr(), n)
    ctx.sync()
    assert len(attn.cache) == n
    pos = np.arange(n)
    for got, pages in zip(attn.cache.export(), (kp, vp)):
        want = pages.float().cpu().numpy()[table.cpu().numpy()[pos // P], :, pos % P].transpose(1, 0, 2)
        assert np.array_equal(got, want)
    paged.gather_dev(attn, kp.data_ptr(), vp.data_ptr(), NP, table.data_ptr(), 0)
    assert len(attn.cache) == 0
    paged.close()
    attn.close()


def test_copy_refusals_and_bad_indexes(ctx):
    import torch
    import shainet_b200 as S
    from shainet_b200 import _lib
    attn = S.LlamaAttention(ctx, 8, 2, 64)
    paged = S.PagedAttention(ctx, 8, 2, 64, 16)
    attn.cache.fill_normal(40, 3)
    kp, vp = (torch.zeros(5, 2, 16, 64, device="cuda") for _ in range(2))
    idx = torch.tensor([0, 1, 80, 3, 2**31 - 1] + [5] * 8, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with pytest.raises(S.ShainetAttnError) as e:
        paged.scatter_dev(attn, kp.data_ptr(), vp.data_ptr(), 5, idx.data_ptr(), 36, 5)
    assert "of a cache of 40" in str(e.value)
    paged.scatter_dev(attn, kp.data_ptr(), vp.data_ptr(), 5, idx.data_ptr(), 0, 5)     # slots 80 and 2^31 - 1 are outside
    with pytest.raises(S.ShainetAttnError) as e:
        ctx.sync()
    assert e.value.code == _lib.E_INVALID
    k, _ = attn.cache.export()
    assert np.array_equal(kp.cpu().numpy()[0, :, [0, 1, 3]], k.transpose(1, 0, 2)[[0, 1, 3]]) and float(kp.abs().sum()) == pytest.approx(
        float(np.abs(k[:, [0, 1, 3]]).sum()), rel=1e-5)
    bad = torch.tensor([0, 5, -1], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    paged.gather_dev(attn, kp.data_ptr(), vp.data_ptr(), 5, bad.data_ptr(), 40)
    with pytest.raises(S.ShainetAttnError):
        ctx.sync()
    # a stream that is being captured cannot grow the cache
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        kp.zero_()
        with pytest.raises(S.ShainetAttnError) as e:
            paged.gather_dev(attn, kp.data_ptr(), vp.data_ptr(), 5, bad.data_ptr(), 100000, stream=stream.cuda_stream)
        assert e.value.code == _lib.E_STATE
    ctx.sync()
    paged.close()
    attn.close()
