"""Calls of the paged operators and the 4-bit products that the documentation allows and that come rarely: the very first call
of a process under stream capture, caches that reserve their addresses, the most rows that a product takes."""
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ctx():
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    yield c
    c.close()


_FIRST = r"""
import sys
sys.path.insert(0, sys.argv[1])
import numpy as np, torch
import shainet_b200 as S
what, ctx = sys.argv[2], S.AttnContext(0)
ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
s = stream.cuda_stream
torch.manual_seed(0)
if what.startswith("q4"):
    M = int(what.split("_")[1])
    p, sc = torch.randint(0, 256, (700, 256), device="cuda", dtype=torch.uint8), torch.rand(700, 8, device="cuda")
    x, y = torch.randn(M, 512, device="cuda"), torch.empty(M, 700, device="cuda")
    torch.cuda.synchronize()
    w = S.Q4Weight.from_device(ctx, p.data_ptr(), sc.data_ptr(), 512, 700, 64)
    call = lambda: w.gemv_dev(x.data_ptr(), y.data_ptr(), M, stream=s)
elif what == "plan":
    a = [ints(5, 0), ints(1, 20), ints(0, -1, -1, -1, -1, -1), ints(1, 2, 3, -1), ints(3), ints(0, 0), ints(0), ints(0, 0, 0), ints(*[0] * 32), ints(9, 9)]
    y = a[8]
    call = lambda: S.plan_pages_dev(ctx, 2, a[0].data_ptr(), a[1].data_ptr(), a[2].data_ptr(), 3, 16, a[3].data_ptr(), 4, a[4].data_ptr(),
                                    a[5].data_ptr(), a[6].data_ptr(), a[7].data_ptr(), a[8].data_ptr(), 32, a[9].data_ptr(), stream=s)
else:
    attn, paged = S.LlamaAttention(ctx, 8, 2, 64, initial_capacity=256), S.PagedAttention(ctx, 8, 2, 64, 16)
    kp, vp = torch.randn(4, 2, 16, 64, device="cuda"), torch.randn(4, 2, 16, 64, device="cuda")
    q, k, v, t, n = torch.randn(512, device="cuda"), torch.randn(128, device="cuda"), torch.randn(128, device="cuda"), ints(2, 0, 1, 3), ints(40)
    if what == "decode":
        y = torch.empty(512, device="cuda")
        call = lambda: paged.decode_dev(attn, kp.data_ptr(), vp.data_ptr(), 4, q.data_ptr(), k.data_ptr(), v.data_ptr(), y.data_ptr(), t.data_ptr(),
                                        4, n.data_ptr(), 1, 0.125, stream=s)
    else:
        class A:
            __cuda_array_interface__ = dict(shape=(2, 256, 64), typestr="<f4", data=(attn.cache.device_ptrs()[0], False), strides=None, version=3)
        y = torch.as_tensor(A(), device="cuda")
        call = lambda: paged.gather_dev(attn, kp.data_ptr(), vp.data_ptr(), 4, t.data_ptr(), 50, stream=s)
torch.cuda.synchronize()
with torch.cuda.graph(graph, stream=stream):
    call()
graph.replay()
torch.cuda.synchronize()
ctx.sync()
got = y.clone()
y.fill_(7)
torch.cuda.synchronize()
call()
torch.cuda.synchronize()
ctx.sync()
same = torch.equal(got[:, :50], y[:, :50]) if what == "gather" else torch.equal(got, y)
print("same" if same and float(got.float().abs().sum()) > 0 else "DIFFERENT")
"""


@pytest.mark.parametrize("what", ["q4_1", "q4_8", "q4_40", "plan", "decode", "gather"])
def test_the_first_call_of_a_process_is_captured(ctx, what):
    """What a kernel's first launch sets up is set up under capture, too."""
    r = subprocess.run([sys.executable, "-c", _FIRST, ROOT, what], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stdout[-500:] + r.stderr[-2000:]


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_copies_of_a_reserved_cache(ctx, kv):
    """Pages are mapped behind the rows as a gather needs them; a token behind it; past the reservation it is refused."""
    import torch
    import shainet_b200 as S
    H, KV, hd, P, n = 8, 2, 128, 16, 9000
    attn = S.LlamaAttention(ctx, H, KV, hd, kv_format=kv, reserve_capacity=10000)
    plain = S.LlamaAttention(ctx, H, KV, hd, kv_format=kv)
    paged = S.PagedAttention(ctx, H, KV, hd, P, kv)
    dt = torch.float32 if kv == "f32" else torch.bfloat16
    NP = -(-n // P)
    kp, vp = (torch.randn(NP, KV, P, hd, device="cuda").to(dt) for _ in range(2))
    row = torch.randperm(NP, device="cuda").to(torch.int32)
    q, k, v = torch.randn(H * hd, device="cuda"), torch.randn(KV * hd, device="cuda"), torch.randn(KV * hd, device="cuda")
    outs = []
    torch.cuda.synchronize()
    for a in (attn, plain):
        for m in (100, n):
            out = torch.full((H * hd,), float("nan"), device="cuda")
            torch.cuda.synchronize()
            paged.gather_dev(a, kp.data_ptr(), vp.data_ptr(), NP, row.data_ptr(), m)
            a.forward_cached_dev(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 1)
            ctx.sync()
            outs.append(out)
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]) and torch.isfinite(outs[1]).all()
    slots = torch.arange(200, dtype=torch.int32, device="cuda")
    k2, v2 = torch.zeros_like(kp), torch.zeros_like(vp)
    torch.cuda.synchronize()
    paged.scatter_dev(attn, k2.data_ptr(), v2.data_ptr(), NP, slots.data_ptr(), 8500, 200)
    ctx.sync()
    pos = torch.arange(8500, 8700, device="cuda")
    assert torch.equal(k2[slots // P, :, slots % P], kp[row[pos // P].long(), :, pos % P])
    assert not k2[13:].any()
    with pytest.raises(S.ShainetAttnError) as e:
        paged.gather_dev(attn, kp.data_ptr(), vp.data_ptr(), NP, row.data_ptr(), attn.cache.capacity + 1)
    assert "reserved" in str(e.value) and len(attn.cache) == n + 1
    for o in (paged, attn, plain):
        o.close()


def test_the_most_rows_of_a_product(ctx):
    import torch
    import shainet_b200 as S
    from shainet_b200 import _lib
    M, K, N = 1 << 20, 64, 24
    rng = np.random.default_rng(1)
    packed = rng.integers(0, 256, (N, K // 2)).astype(np.uint8)
    scales = np.float32(2.0) ** rng.integers(-3, 4, (N, 1)).astype(np.float32)
    W = S.Q4Weight.from_quantized(ctx, packed, scales, K, 64)
    x = torch.randint(-8, 9, (M + 4, K), device="cuda").float()
    y = torch.full((M + 4, N), float("nan"), device="cuda")
    torch.cuda.synchronize()
    W.gemv_dev(x.data_ptr(), y.data_ptr(), M)
    ctx.sync()
    q = np.stack([packed & 15, packed >> 4], -1).reshape(N, K).astype(np.float32) - 8
    want = x[:M].double() @ torch.from_numpy(q * scales).cuda().double().T
    assert torch.equal(y[:M].double(), want) and torch.isnan(y[M:]).all()          # every sum is exact in fp32
    with pytest.raises(S.ShainetAttnError) as e:
        W.gemv_dev(x.data_ptr(), y.data_ptr(), M + 1)
    assert e.value.code == _lib.E_UNSUPPORTED
    W.close()
