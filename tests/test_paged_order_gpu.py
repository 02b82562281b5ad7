"""Order of calls on one stream and on several: a decode token straight behind the copy that filled its cache from pages.  The
launch may start while the copy ends; it must see every row of it.  And decode tokens of one sequence with calls of the same
context on another stream in between, which say nothing about the row that the token before still appends.  Outputs are compared bit for bit with the same calls
that wait for each other on the host."""
import numpy as np
import pytest

from helpers import DECODE_TOL, L1B, Q30, Q8B, rel_err

pytestmark = pytest.mark.gpu
SHAPES = {"L1B": L1B, "Q8B": Q8B, "Q30": Q30, "g16": dict(H=32, KV=2, hd=128, theta=1e6), "g7": dict(H=28, KV=4, hd=128, theta=1e6)}


@pytest.fixture(scope="module")
def ctx():
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    yield c
    c.close()


class Turns:
    """Two requests in pages whose rows differ, and a contiguous cache that takes one or the other."""

    def __init__(self, ctx, sh, n, P, kv, seed=3):
        import torch
        import shainet_b200 as S
        self.ctx, self.torch, self.n, self.P = ctx, torch, n, P
        self.H, self.KV, self.hd = sh["H"], sh["KV"], sh["hd"]
        dt = torch.float32 if kv == "f32" else torch.bfloat16
        gen = torch.Generator("cuda").manual_seed(seed)
        per = -(-(n + 1) // P)
        self.NP = 2 * per + 1
        self.kp, self.vp = (torch.randn(self.NP, self.KV, P, self.hd, generator=gen, device="cuda").to(dt) for _ in range(2))
        order = torch.randperm(self.NP, generator=gen, device="cuda").to(torch.int32)
        self.rows = [order[:per].contiguous(), order[per:2 * per].contiguous()]
        self.q, self.k, self.v = (torch.randn(m * self.hd, generator=gen, device="cuda") for m in (self.H, self.KV, self.KV))
        self.attn = S.LlamaAttention(ctx, self.H, self.KV, self.hd, sh["theta"], kv_format=kv, initial_capacity=n + 300)
        self.paged = S.PagedAttention(ctx, self.H, self.KV, self.hd, P, kv)
        self.stream = torch.cuda.Stream()
        torch.cuda.synchronize()

    def gather(self, which, attn=None, n=None):
        self.paged.gather_dev(attn or self.attn, self.kp.data_ptr(), self.vp.data_ptr(), self.NP, self.rows[which].data_ptr(),
                              self.n if n is None else n, stream=self.stream.cuda_stream)

    def token(self, out, flags=0):
        self.attn.forward_cached_dev(self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), out.data_ptr(), 1,
                                     stream=self.stream.cuda_stream, flags=flags)

    def new(self):
        out = self.torch.full((self.H * self.hd,), float("nan"), device="cuda")
        self.torch.cuda.synchronize()
        return out

    def wait(self):
        self.torch.cuda.synchronize()
        self.ctx.sync()

    def close(self):
        self.paged.close()
        self.attn.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("shape,n,P", [("L1B", 1, 16), ("L1B", 45, 16), ("L1B", 4000, 16), ("Q8B", 900, 24), ("Q8B", 9001, 64), ("Q30", 20000, 128),
                                       ("g16", 700, 16), ("g7", 700, 16)])
def test_a_token_straight_behind_the_rows(ctx, shape, n, P, kv):
    """Gather of one request, one token; of the other, one token; two tokens behind one gather; the rows of the last turn in
    the cache are another request's every time."""
    import shainet_b200 as S
    t = Turns(ctx, SHAPES[shape], n, P, kv)
    want = []
    for which in (0, 1):
        t.gather(which)
        t.wait()
        one, two = t.new(), t.new()
        t.token(one)
        t.wait()
        t.token(two)
        t.wait()
        want.append((one, two))
    assert not t.torch.equal(want[0][0], want[1][0])
    for flags in (0, S.F_INPUTS_READY):
        outs = [(t.new(), t.new()) for _ in range(20)]
        for i, (one, two) in enumerate(outs):
            t.gather(i & 1)
            t.token(one, flags)
            t.token(two)
        t.wait()
        for i, (one, two) in enumerate(outs):
            assert t.torch.equal(one, want[i & 1][0]) and t.torch.equal(two, want[i & 1][1]), i
    t.close()


def test_the_same_rows_as_a_decode_over_the_pages(ctx):
    """The turn's output is that of the paged decode of the same request, to the sum of both sides' fp32 decode classes."""
    t = Turns(ctx, dict(L1B, theta=5e5), 1234, 16, "f32")
    import torch
    out, ref = t.new(), t.new()
    t.gather(1)
    t.token(out)
    lens = torch.tensor([t.n + 1], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    t.paged.decode_dev(t.attn, t.kp.data_ptr(), t.vp.data_ptr(), t.NP, t.q.data_ptr(), t.k.data_ptr(), t.v.data_ptr(), ref.data_ptr(),
                       t.rows[1].data_ptr(), len(t.rows[1]), lens.data_ptr(), 1, t.attn.scale, stream=t.stream.cuda_stream)
    t.wait()
    assert rel_err(out.cpu().numpy(), ref.cpu().numpy()) <= 2 * DECODE_TOL
    t.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_a_batch_with_one_refilled_cache(ctx, kv):
    import shainet_b200 as S
    t = Turns(ctx, SHAPES["Q8B"], 3000, 16, kv)
    torch = t.torch
    others = [S.LlamaAttention(ctx, t.H, t.KV, t.hd, SHAPES["Q8B"]["theta"], kv_format=kv) for _ in range(2)]
    for i, o in enumerate(others):
        o.cache.fill_normal(500 + 700 * i, 7 + i)
    q, k, v = (torch.randn(3, m * t.hd, device="cuda") for m in (t.H, t.KV, t.KV))

    def step(wait, which):
        out = torch.full((3, t.H * t.hd), float("nan"), device="cuda")
        torch.cuda.synchronize()
        t.gather(which)
        if wait:
            t.wait()
        S.forward_batched_dev(ctx, [others[0].cache, t.attn.cache, others[1].cache], q.data_ptr(), k.data_ptr(), v.data_ptr(),
                              out.data_ptr(), t.attn.scale, stream=t.stream.cuda_stream)
        for o in others:
            o.cache.truncate(len(o.cache) - 1)
        return out

    want = [step(True, w) for w in (0, 1)]
    got = [step(False, i & 1) for i in range(20)]
    t.wait()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i & 1]), i
    for o in others:
        o.close()
    t.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_tokens_behind_replays_of_a_captured_copy(ctx, kv):
    """A graph fills the cache, an eager token follows, over and over: the graph's copies are not seen by the host."""
    import torch
    import shainet_b200 as S
    t = Turns(ctx, SHAPES["Q8B"], 2500, 16, kv)
    want, graphs = [], [torch.cuda.CUDAGraph() for _ in range(2)]
    for which in (0, 1):
        t.gather(which)
        t.wait()
        want.append(t.new())
        t.token(want[-1])
        t.wait()
        with torch.cuda.graph(graphs[which], stream=t.stream):
            t.gather(which)
    outs = [t.new() for _ in range(40)]
    with torch.cuda.stream(t.stream):
        for i, out in enumerate(outs):
            t.attn.cache.truncate(2500)
            graphs[i & 1].replay()
            t.token(out, S.F_INPUTS_READY if i & 2 else 0)
    t.wait()
    for i, out in enumerate(outs):
        assert torch.equal(out, want[i & 1]), i
    del graphs
    t.close()


def test_an_emptied_cache_starts_again(ctx):
    t = Turns(ctx, SHAPES["L1B"], 64, 16, "f32")
    out, ref = t.new(), t.new()
    t.gather(0)
    t.token(out)
    t.gather(0, n=0)
    assert len(t.attn.cache) == 0
    t.token(out)
    t.wait()
    t.attn.clear_cache()
    t.token(ref)
    t.wait()
    assert t.torch.equal(out, ref) and len(t.attn.cache) == 1
    t.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("between", ["q4", "q4_rows", "plan", "paged_decode"])
def test_tokens_of_one_sequence_with_calls_on_another_stream_between(ctx, between, kv):
    """Token, a call elsewhere, token, ...: every token sees the row of the one before it.  The rows are large against what
    else the sequence holds, so that a row read too early (what an earlier round left there, times minus one) shows."""
    import torch
    import shainet_b200 as S
    sh, n, steps = SHAPES["L1B"], 37, 60
    H, KV, hd = sh["H"], sh["KV"], sh["hd"]
    attn = S.LlamaAttention(ctx, H, KV, hd, sh["theta"], kv_format=kv, initial_capacity=512)
    side = S.LlamaAttention(ctx, H, KV, hd, sh["theta"], kv_format=kv)      # gives the paged decode its parameters
    paged = S.PagedAttention(ctx, H, KV, hd, 16, kv)
    rng = np.random.default_rng(4)
    W = S.Q4Weight.from_simple(ctx, rng.standard_normal((256, 512)).astype(np.float32), 64)
    gen = torch.Generator("cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, y = r(40, 256), torch.empty(40, 512, device="cuda")
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    lens, delta, table, free, count = ints(5), ints(1), ints(0, 1, -1), ints(2, 3, -1, -1), ints(2)
    lo, co, first, slots, status = ints(0), ints(0), ints(0, 0), ints(0, 0, 0, 0), ints(0, 0)
    dt = torch.float32 if kv == "f32" else torch.bfloat16
    kp, vp = r(4, KV, 16, hd).to(dt), r(4, KV, 16, hd).to(dt)
    sq, sk, sv, so = r(H * hd), r(KV * hd), r(KV * hd), torch.empty(H * hd, device="cuda")
    q, k, v = r(steps, H * hd), r(steps, KV * hd), 3.0 * r(steps, KV * hd)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()

    def elsewhere():
        s = b.cuda_stream
        if between in ("q4", "q4_rows"):
            W.gemv_dev(x.data_ptr(), y.data_ptr(), 1 if between == "q4" else 40, stream=s)
        if between == "plan":
            S.plan_pages_dev(ctx, 1, lens.data_ptr(), delta.data_ptr(), table.data_ptr(), 3, 16, free.data_ptr(), 4, count.data_ptr(),
                             lo.data_ptr(), co.data_ptr(), first.data_ptr(), slots.data_ptr(), 4, status.data_ptr(), stream=s)
        if between == "paged_decode":
            paged.decode_dev(side, kp.data_ptr(), vp.data_ptr(), 4, sq.data_ptr(), sk.data_ptr(), sv.data_ptr(), so.data_ptr(),
                             table.data_ptr(), 3, lens.data_ptr(), 1, 0.125, stream=s)

    def round_(sign, wait, flags=0):
        attn.clear_cache()
        attn.cache.fill_normal(n, 6)
        vs = (sign * v).contiguous()
        out = torch.full((steps, H * hd), float("nan"), device="cuda")
        torch.cuda.synchronize()
        for i in range(steps):
            attn.forward_cached_dev(q[i].data_ptr(), k[i].data_ptr(), vs[i].data_ptr(), out[i].data_ptr(), 1, stream=a.cuda_stream,
                                    flags=flags)
            if wait:
                torch.cuda.synchronize()
            else:
                elsewhere()
        torch.cuda.synchronize()
        ctx.sync()
        return out

    want = {s: round_(s, True) for s in (1.0, -1.0)}
    for rep in range(8):
        for s in (1.0, -1.0):
            assert torch.equal(round_(s, False), want[s]), (rep, s)
            assert torch.equal(round_(s, False, S.F_INPUTS_READY), want[s]), (rep, s)
    for o in (W, paged, side, attn):
        o.close()
