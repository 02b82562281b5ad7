"""Attention over pages where one request's visible rows or projections are not finite: the others' outputs and pages are,
bit for bit, what they are without it.  The requests share the line of tiles, so the CTAs that work on the bad one also work on
its neighbours.  And batches that name more rows than there can be."""
import numpy as np
import pytest

from test_paged_decode_gpu import LAYOUTS, Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    yield c
    c.close()


def bits(x):
    return np.ascontiguousarray(x).view(np.uint32)


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("layout,lens", [("L1B", [700, 3, 900, 0, 33, 1500]), ("mha", [100, 40, 700, 1, 0, 64]), ("Q30", [20, 5000, 9000, 17, 300, 1]),
                                         ("g16", [33, 1, 2000, 700, 0, 90]), ("g40", [50, 70, 300, 0, 16, 800])])
def test_one_bad_request_leaves_the_others_alone(ctx, layout, lens, kv):
    import torch
    b = Batch(ctx, LAYOUTS[layout], lens, 16, kv, 41)
    clean = b.run()
    bad, others = 2, [0, 1, 3, 4, 5]
    n, hd, KV = lens[bad], b.sh["hd"], b.sh["KV"]
    own_pages = set(int(p) for p in b.table[bad, :-(-n // 16)])
    keep = np.array([p not in own_pages for p in range(b.NP)])
    at = lambda pos: (int(b.table[bad, pos // 16]), slice(None), pos % 16)
    for value in (float("nan"), float("inf"), float("-inf")):
        for what in ("k", "v", "q", "k_new", "v_new", "all_k"):
            # as before the first call: its rows, its inputs
            b.tk.copy_(torch.from_numpy(b.k)), b.tv.copy_(torch.from_numpy(b.v))
            b.tq.copy_(torch.from_numpy(b.q)), b.tkn.copy_(torch.from_numpy(b.kn)), b.tvn.copy_(torch.from_numpy(b.vn))
            if what == "k": b.tk[at(n // 3)][:, hd // 2] = value
            if what == "v": b.tv[at(n // 2)] = value
            if what == "q": b.tq[bad, 5] = value
            if what == "k_new": b.tkn[bad] = value
            if what == "v_new": b.tvn[bad, -1] = value
            if what == "all_k":
                for p in own_pages:
                    b.tk[p] = value
            b.out.fill_(float("nan"))
            torch.cuda.synchronize()
            got = b.run()
            assert np.array_equal(bits(got[0][others]), bits(clean[0][others])), (value, what)
            for g, c in zip(got[1:], clean[1:]):
                assert np.array_equal(g[keep], c[keep], equal_nan=True), (value, what)
    b.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_more_rows_than_there_can_be(ctx, kv):
    """Tables that name the same pages over and over: 2^31 - 1 positions of one request, and 999 of sixteen million each,
    are more than the line of tiles holds.  All rows are zeros, no page is written, the call says so and the next one works."""
    import torch
    import shainet_b200 as S
    from shainet_b200 import _lib
    H, KV, hd, P = 16, 8, 128, 4096
    attn, paged = S.LlamaAttention(ctx, H, KV, hd, kv_format=kv), S.PagedAttention(ctx, H, KV, hd, P, kv)
    dt = torch.float32 if kv == "f32" else torch.bfloat16
    kp, vp = (torch.randn(2, KV, P, hd, device="cuda").to(dt) for _ in range(2))
    before = kp.clone(), vp.clone()
    for R, W, lens in ((2, 1 << 19, [2**31 - 1, 5]), (1000, 4096, [16000000] * 999 + [7])):
        table = torch.zeros(R, W, dtype=torch.int32, device="cuda")
        q, k, v = (torch.randn(R, n * hd, device="cuda") for n in (H, KV, KV))
        out = torch.full((R, H * hd), float("nan"), device="cuda")
        tl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        call = lambda: paged.decode_dev(attn, kp.data_ptr(), vp.data_ptr(), 2, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                        table.data_ptr(), W, tl.data_ptr(), R, 0.1)
        torch.cuda.synchronize()
        call()
        with pytest.raises(S.ShainetAttnError) as e:
            ctx.sync()
        assert e.value.code == _lib.E_INVALID
        assert not out.any() and torch.equal(kp, before[0]) and torch.equal(vp, before[1])
        tl.zero_()
        tl[1] = 3
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        call()
        ctx.sync()
        assert out[1].isfinite().all() and out[1].any() and not out[0].any()
        for x, y in zip((kp, vp), before):
            x.copy_(y)
    paged.close()
    attn.close()
