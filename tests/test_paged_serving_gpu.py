"""The paged operators together, as a server uses them: page plans, 4-bit projections, attention over pages, prompts that run
on a contiguous cache and move into pages, a second turn that comes back from them, requests that finish and make room.  One
attention layer (projections, attention, output projection with the residual added outside); beside it the same steps run on
one contiguous cache per request through the framework's existing entries, in fp32 or bfloat16 rows.

Both sides compute the same function with fp32 sums in another order: outputs agree within twice DECODE_TOL (each side's
own), prompt rows within the TF32 prefill class on both sides alike, as the rows are copied and not recomputed.

With 16-bit rows the two sides' new rows may differ by a flip: a projection of four rows and one of a single row add in another
order, and an element within 2^-24 of the middle between two bfloat16 values is rounded up on one side and down on the other,
a difference of one spacing, at most 2^-7 of the element.  In a v row that changes an output by p 2^-7 |v|, in a k row it
changes the row's score by scale |q| 2^-7 |k|, with |q|, |k| up to 4 and scale 1/8 by 1.6e-2, and the outputs by p 1.6e-2 |v|
at most, where p is the row's weight: below 0.3 here (17 positions or more of scores within +-3, or rows that only this step
saw).  0.3 x 1.6e-2 = 4.8e-3 of the largest value: BF16_TOL = 5e-3, the tolerance of the framework's other tests that meet
such flips."""
import numpy as np
import pytest

from helpers import DECODE_TOL, rel_err

pytestmark = pytest.mark.gpu
H, KV, HD, D, P = 8, 2, 64, 512, 16
BF16_TOL = 5e-3
THETA = 500000.0


@pytest.fixture(scope="module")
def ctx():
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    yield c
    c.close()


class Layer:
    def __init__(self, ctx, kv, seed, requests, num_pages, width):
        import torch
        import shainet_b200 as S
        self.ctx, self.S, self.kv, self.torch = ctx, S, kv, torch
        rng = self.rng = np.random.default_rng(seed)
        w = lambda K, N: S.Q4Weight.from_simple(ctx, (rng.standard_normal((K, N)) / np.sqrt(K)).astype(np.float32), 64)
        self.wq, self.wk, self.wv, self.wo = w(D, H * HD), w(D, KV * HD), w(D, KV * HD), w(H * HD, D)
        self.attn = S.LlamaAttention(ctx, H, KV, HD, THETA, kv_format=kv)      # prompts run here, one after another
        self.paged = S.PagedAttention(ctx, H, KV, HD, P, kv)
        self.alone = [S.LlamaAttention(ctx, H, KV, HD, THETA, kv_format=kv) for _ in range(requests)]
        dt = torch.float32 if kv == "f32" else torch.bfloat16
        self.pages = [torch.full((num_pages, KV, P, HD), float("nan"), dtype=dt, device="cuda") for _ in range(2)]
        ints = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
        self.R, self.W, self.NP, self.tokens = requests, width, num_pages, 256
        self.lens, self.delta, self.table, self.count = ints(requests), ints(requests), ints(requests, width), ints(1)
        self.free, self.first, self.slots, self.status = ints(num_pages), ints(requests + 1), ints(self.tokens), ints(2)
        self.free.copy_(torch.from_numpy(rng.permutation(num_pages).astype(np.int32)))
        self.count.fill_(num_pages)
        torch.cuda.synchronize()
        self.stream = torch.cuda.current_stream().cuda_stream

    def plan(self, delta):
        self.delta.copy_(self.torch.tensor(delta, dtype=self.torch.int32))
        self.S.plan_pages_dev(self.ctx, self.R, self.lens.data_ptr(), self.delta.data_ptr(), self.table.data_ptr(), self.W, P,
                              self.free.data_ptr(), self.NP, self.count.data_ptr(), self.lens.data_ptr(), self.count.data_ptr(),
                              self.first.data_ptr(), self.slots.data_ptr(), self.tokens, self.status.data_ptr(), stream=self.stream)

    def rows(self, x):
        """Projected rows of activations [n, D]."""
        out = []
        for w in (self.wq, self.wk, self.wv):
            y = self.torch.empty(len(x), w.N, device="cuda")
            w.gemv_dev(x.data_ptr(), y.data_ptr(), len(x), stream=self.stream)
            out.append(y)
        return out

    def output(self, y):
        out = self.torch.empty(len(y), D, device="cuda")
        self.wo.gemv_dev(y.data_ptr(), out.data_ptr(), len(y), stream=self.stream)
        return out

    def prompt(self, r, x, old=0):
        """Activations of new positions of request r behind `old` ones: run on the contiguous cache, move into the pages that
        the plan just made."""
        q, k, v = self.rows(x)
        n = len(x)
        y = self.torch.empty_like(q)
        pages = [t.data_ptr() for t in self.pages]
        if old:
            self.paged.gather_dev(self.attn, *pages, self.NP, self.table[r].data_ptr(), old, stream=self.stream)
        else:
            self.torch.cuda.synchronize()
            self.attn.clear_cache()
        self.attn.forward_cached_dev(q.data_ptr(), k.data_ptr(), v.data_ptr(), y.data_ptr(), n, stream=self.stream)
        first = int(self.first[r])
        self.paged.scatter_dev(self.attn, *pages, self.NP, self.slots[first:].data_ptr(), old, n, stream=self.stream)
        return self.output(y)

    def decode(self, x):
        q, k, v = self.rows(x)
        y = self.torch.empty_like(q)
        pages = [t.data_ptr() for t in self.pages]
        self.paged.decode_dev(self.attn, *pages, self.NP, q.data_ptr(), k.data_ptr(), v.data_ptr(), y.data_ptr(), self.table.data_ptr(),
                              self.W, self.lens.data_ptr(), self.R, self.attn.scale, stream=self.stream)
        return self.output(y)

    def alone_step(self, r, x):
        """The same rows of one request on its own contiguous cache."""
        q, k, v = self.rows(x)
        y = self.torch.empty_like(q)
        self.torch.cuda.synchronize()
        self.alone[r].forward_cached_dev(q.data_ptr(), k.data_ptr(), v.data_ptr(), y.data_ptr(), len(x), stream=self.stream)
        return self.output(y)

    def check(self, got, want):
        self.torch.cuda.synchronize()
        self.ctx.sync()
        assert rel_err(got.cpu().numpy(), want.cpu().numpy()) <= (2 * DECODE_TOL if self.kv == "f32" else BF16_TOL)

    def close(self):
        for o in (self.paged, self.attn, *self.alone, self.wq, self.wk, self.wv, self.wo):
            o.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_a_server_in_small(ctx, kv):
    import torch
    L = Layer(ctx, kv, 5, requests=4, num_pages=40, width=20)
    act = lambda n: torch.from_numpy(L.rng.standard_normal((n, D)).astype(np.float32)).cuda()
    held = [0, 0, 0, 0]

    def start(r, n):
        delta = [0] * 4
        delta[r] = n
        L.plan(delta)
        x = act(n)
        L.check(L.prompt(r, x, held[r]), L.alone_step(r, x))
        held[r] += n

    def step():
        """One decode token for every request that holds something; the others are padded rows."""
        L.plan([1 if n else 0 for n in held])
        x = act(4)
        got = L.decode(x)
        for r, n in enumerate(held):
            if n:
                L.check(got[r:r + 1], L.alone_step(r, x[r:r + 1]))
                held[r] += 1
            else:
                assert not got[r].any()

    start(0, 100)                      # tensor-core prompt
    start(2, 17)                       # a few rows over one page
    for _ in range(20):
        step()
    start(2, 5)                        # a second turn over what is in the pages
    start(1, 200)
    for _ in range(3):
        step()
    assert L.lens.tolist() == held and L.status.tolist() == [0, 0]
    assert int(L.count[0]) == 40 - sum(-(-n // P) for n in held)
    # request 0 is done, request 1 takes back a draft of 9 positions, request 3 needs the room
    L.plan([-held[0], -9, 0, 0])
    L.alone[0].clear_cache()
    L.alone[1].cache.truncate(held[1] - 9)
    held[0], held[1] = 0, held[1] - 9
    start(3, 130)
    for _ in range(18):
        step()
    assert L.lens.tolist() == held
    # more than there is: nothing changes, and the next step goes on
    before = [t.clone() for t in (L.lens, L.table, L.free, L.count)]
    L.plan([300, 0, 0, 0])
    torch.cuda.synchronize()
    assert L.status.tolist()[0] != 0 and all(torch.equal(a, b) for a, b in zip(before, (L.lens, L.table, L.free, L.count)))
    step()
    L.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_decode_loop_as_one_graph(ctx, kv):
    """Plan, projections, attention and output projection captured once; the lengths advance on the device, across page
    borders.  The same steps without a graph on a second state give the same bits."""
    import torch
    runs = []
    for captured in (False, True):
        L = Layer(ctx, kv, 6, requests=4, num_pages=40, width=20)
        torch.manual_seed(1)
        for r, n in ((0, 31), (1, 90), (3, 1)):
            delta = [0] * 4
            delta[r] = n
            L.plan(delta)
            L.prompt(r, torch.randn(n, D).cuda())
        xs, delta = torch.randn(24, 4, D).cuda(), torch.tensor([1, 1, 0, 1], dtype=torch.int32).cuda()
        x, outs = torch.empty(4, D, device="cuda"), []

        def once():
            L.S.plan_pages_dev(ctx, 4, L.lens.data_ptr(), delta.data_ptr(), L.table.data_ptr(), L.W, P, L.free.data_ptr(), L.NP,
                               L.count.data_ptr(), L.lens.data_ptr(), L.count.data_ptr(), L.first.data_ptr(), L.slots.data_ptr(),
                               L.tokens, L.status.data_ptr(), stream=L.stream)
            return L.decode(x)

        torch.cuda.synchronize()
        if captured:
            stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
            L.stream = stream.cuda_stream
            with torch.cuda.graph(graph, stream=stream):
                y = once()
        for i in range(24):
            x.copy_(xs[i])
            torch.cuda.synchronize()
            if captured:
                graph.replay()
            else:
                y = once()
            torch.cuda.synchronize()
            outs.append(y.cpu().numpy().copy())
        ctx.sync()
        assert L.lens.tolist() == [55, 114, 0, 25]
        runs.append(np.stack(outs))
        if captured:
            del graph
        L.close()
    assert np.array_equal(runs[0], runs[1]) and not runs[0][:, 2].any() and np.isfinite(runs[0]).all()
