"""Page plans and the decode of the same step: the lengths that the plan writes for it, and captured loops of both in which
requests idle, shrink, start, end, or a step cannot be taken.  Lengths and pages are compared for equality, outputs bit for
bit with a decode over the same lengths made by the host."""
import numpy as np
import pytest

from test_paged_plan_gpu import host_plan, mixed, state

pytestmark = pytest.mark.gpu
H, KV, HD = 8, 2, 64


@pytest.fixture(scope="module")
def ctx():
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    yield c
    c.close()


def dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


def step(ctx, lens, delta, table, P, free, count, tokens, in_place):
    """(status, decode_lens, everything else) of one step on the device."""
    import torch
    import shainet_b200 as S
    tl, td, tt, tf, tc = dev(lens), dev(delta), dev(table), dev(free), dev([count])
    lo, co = (tl, tc) if in_place else (torch.full_like(tl, -5), torch.full_like(tc, -5))
    R = len(lens)
    first, slots, status = dev(np.full(R + 1, -5)), dev(np.full(tokens, -5)), dev([-5, -5])
    dl = dev(np.full(R + 3, -5))
    torch.cuda.synchronize()
    S.plan_pages_dev(ctx, R, tl.data_ptr(), td.data_ptr(), tt.data_ptr(), table.shape[1], P, tf.data_ptr(), len(free), tc.data_ptr(),
                     lo.data_ptr(), co.data_ptr(), first.data_ptr(), slots.data_ptr(), tokens, status.data_ptr(),
                     decode_lens_ptr=dl.data_ptr())
    ctx.sync()
    assert (dl[R:] == -5).all()
    rest = [lo.cpu().numpy(), int(co[0]), tt.cpu().numpy(), tf.cpu().numpy(), first.cpu().numpy(), slots.cpu().numpy()]
    return status.tolist(), dl[:R].cpu().numpy(), rest


@pytest.mark.parametrize("in_place", [False, True], ids=["out", "in_place"])
@pytest.mark.parametrize("R,P,longest", [(1, 16, 40), (7, 24, 100), (64, 16, 30), (256, 32, 700), (2500, 16, 20)])
def test_lengths_for_the_decode(ctx, R, P, longest, in_place):
    """One token: the length with it.  Anything else: 0; the other arrays are those of a step without them.  Then the same
    step one page short, and with a length that cannot be: 0 for all."""
    rng = np.random.default_rng(R + P)
    lens, delta = mixed(rng, R, P, longest)
    delta[0] = 1
    W = int(max(np.maximum(lens, lens + delta).max(), 1) + P - 1) // P + 2
    held, after = (lens + P - 1) // P, (lens + delta + P - 1) // P
    need = int(np.maximum(after - held, 0).sum() - np.maximum(held - after, 0).sum())
    spare = max(need, 0)
    table, free = state(rng, R, W, P, int(held.sum()) + spare + 4, lens, spare)
    tokens = int(np.maximum(delta, 0).sum()) + 5
    want = host_plan(lens, delta, table, P, free, spare, tokens)
    status, dl, rest = step(ctx, lens, delta, table, P, free, spare, tokens, in_place)
    assert status == [0, 0] == want[0]
    assert np.array_equal(dl, np.where(delta == 1, lens + 1, 0))
    assert all(np.array_equal(np.asarray(w), np.asarray(g)) for w, g in zip(want[1:], rest))
    bad = lens.copy()
    bad[R // 2] = W * P + 1
    for l, c in ((lens, spare - 1 if need > 0 else None), (bad, spare)):
        if c is None:
            continue
        want = host_plan(l, delta, table, P, free, c, tokens)
        status, dl, rest = step(ctx, l, delta, table, P, free, c, tokens, in_place)
        assert status == want[0] and status[0] != 0 and not dl.any()
        assert all(np.array_equal(np.asarray(w), np.asarray(g)) for w, g in zip(want[1:], rest))


def test_no_requests(ctx):
    empty, free = np.zeros(0, np.int32), np.arange(4, dtype=np.int32)
    status, dl, rest = step(ctx, empty, empty, np.zeros((0, 3), np.int32), 16, free, 4, 5, False)
    assert status == [0, 0] and len(dl) == 0 and (rest[-1] == -1).all()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_captured_loop_writes_only_what_a_step_decodes(ctx, kv):
    """Plan and decode in one graph, replayed.  Steps: all decode; one idles, one gives back a draft, one starts with a prompt of
    seven; one that the pool has no room for; one that ends a request; all decode again.  After each, the pages hold what
    they held but for the rows of the requests that took one token, a request without one has a row of zeros, and the
    outputs are those of a decode over lengths made here."""
    import torch
    import shainet_b200 as S
    rng = np.random.default_rng(11)
    P, W, NP, R, tokens = 8, 12, 40, 5, 128
    lens = np.array([30, 41, 16, 1, 0], np.int32)
    table, free = state(rng, R, W, P, NP, lens, 12)
    count = 12
    dt = torch.float32 if kv == "f32" else torch.bfloat16
    attn = S.LlamaAttention(ctx, H, KV, HD, 1e4, kv_format=kv)
    paged, other = (S.PagedAttention(ctx, H, KV, HD, P, kv) for _ in range(2))
    kp, vp = (torch.randn(NP, KV, P, HD, generator=torch.Generator().manual_seed(i)).to(dt).cuda() for i in range(2))
    q, k, v = (torch.randn(R, n * HD, device="cuda") for n in (H, KV, KV))
    out, ref = (torch.full((R, H * HD), float("nan"), device="cuda") for _ in range(2))
    tl, td, tt, tf, tc = dev(lens), dev(np.zeros(R)), dev(table), dev(free), dev([count])
    first, slots, status, dl = dev(np.zeros(R + 1)), dev(np.zeros(tokens)), dev([9, 9]), dev(np.full(R, -5))
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def decode(handle, kp, vp, lens_t, out_t, s=None):
        handle.decode_dev(attn, kp.data_ptr(), vp.data_ptr(), NP, q.data_ptr(), k.data_ptr(), v.data_ptr(), out_t.data_ptr(),
                          tt.data_ptr(), W, lens_t.data_ptr(), R, 0.125, stream=s)

    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        S.plan_pages_dev(ctx, R, tl.data_ptr(), td.data_ptr(), tt.data_ptr(), W, P, tf.data_ptr(), NP, tc.data_ptr(), tl.data_ptr(),
                         tc.data_ptr(), first.data_ptr(), slots.data_ptr(), tokens, status.data_ptr(), stream=stream.cuda_stream,
                         decode_lens_ptr=dl.data_ptr())
        decode(paged, kp, vp, dl, out, stream.cuda_stream)
    steps = [[1, 1, 1, 1, 0], [1, 0, -5, 1, 7], [1, 50, 1, 1, 60], [1, 1, 0, -3, 1], [1, 1, 1, 0, 1]]
    taken = []
    for delta in steps:
        delta = np.array(delta, np.int32)
        td.copy_(dev(delta))
        for x in (q, k, v):
            x.normal_()
        before = kp.clone(), vp.clone()
        want = host_plan(lens, delta, table, P, free, count, tokens)
        ok = want[0][0] == 0
        taken.append(ok)
        host_lens = np.where((delta == 1) & ok, lens + 1, 0).astype(np.int32)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ctx.sync()
        assert status.tolist() == want[0] and np.array_equal(dl.cpu().numpy(), host_lens)
        _, lens, count, table, free = want[:5]
        assert np.array_equal(tl.cpu().numpy(), lens) and np.array_equal(tt.cpu().numpy(), table)
        decode(other, *before, dev(host_lens), ref)
        torch.cuda.synchronize()
        ctx.sync()
        assert torch.equal(out, ref) and not out[torch.from_numpy(host_lens == 0)].any()
        assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])
    assert taken == [True, True, False, True, True]
    for o in (paged, other, attn):
        o.close()


def test_a_refused_step_leaves_every_row(ctx):
    """The rows of the last positions stay as they were, bit for bit, when the pool is short."""
    import torch
    import shainet_b200 as S
    rng = np.random.default_rng(12)
    P, W, NP, R = 8, 6, 9, 3
    lens, delta = np.array([8, 20, 16], np.int32), np.ones(3, np.int32)
    table, free = state(rng, R, W, P, NP, lens, 1)          # two requests need a page, one is free
    attn, paged = S.LlamaAttention(ctx, H, KV, HD), S.PagedAttention(ctx, H, KV, HD, P)
    kp, vp = (torch.randn(NP, KV, P, HD, device="cuda") for _ in range(2))
    q, k, v = (torch.randn(R, n * HD, device="cuda") for n in (H, KV, KV))
    out = torch.full((R, H * HD), float("nan"), device="cuda")
    tl, td, tt, tf, tc = dev(lens), dev(delta), dev(table), dev(free), dev([1])
    first, slots, status, dl = dev(np.zeros(R + 1)), dev(np.zeros(4)), dev([9, 9]), dev(np.full(R, -5))
    before = kp.clone(), vp.clone()
    torch.cuda.synchronize()
    S.plan_pages_dev(ctx, R, tl.data_ptr(), td.data_ptr(), tt.data_ptr(), W, P, tf.data_ptr(), NP, tc.data_ptr(), tl.data_ptr(),
                     tc.data_ptr(), first.data_ptr(), slots.data_ptr(), 4, status.data_ptr(), decode_lens_ptr=dl.data_ptr())
    paged.decode_dev(attn, kp.data_ptr(), vp.data_ptr(), NP, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), tt.data_ptr(), W,
                     dl.data_ptr(), R, 0.125)
    ctx.sync()
    assert status.tolist() == [1, 1] and dl.tolist() == [0, 0, 0] and tl.tolist() == lens.tolist()
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1]) and not out.any()
    paged.close()
    attn.close()
