"""Timed cases of the operators that serve a batch of requests whose keys and values lie in pages, and of the 4-bit
products around them.

* ``plan``     block tables and slot maps built on the GPU from request lengths (``plan_pages_dev``)
* ``decode``   attention of one new token per request over the pages, with the bias, per-head norm, RoPE and append in
               front of it (``PagedAttention.decode_dev``)
* ``scatter``  rows of a contiguous cache into pages through a slot map (``PagedAttention.scatter_dev``)
* ``gather``   the rows of one request out of its pages into a contiguous cache (``PagedAttention.gather_dev``)
* ``q4``       products of activation rows with 4-bit weights and group scales (``Q4Weight.gemv_dev``)

With ``own`` false ``run`` computes the same in elementary torch operations.
"""
import math
import random

import torch

own = False

# (query heads, kv heads, head_dim, RoPE theta, per-head q/k norm, projection biases)
HEADS = {
    "llama_1b": (32, 8, 64, 500000.0, False, False),
    "qwen3_8b": (32, 8, 128, 1e6, True, False),
    "qwen3_30b": (32, 4, 128, 1e6, True, False),
    "mha_16x64": (16, 16, 64, 10000.0, False, False),       # one query head per kv head
    "gqa_28x4": (28, 4, 128, 1e6, False, True),             # seven query heads per kv head, biased projections
    "mqa_32x2": (32, 2, 128, 1e6, False, False),            # sixteen query heads per kv head
}
EPS = 1e-6


def listed():
    return [
        # The smallest call of a serving loop: eight chats take one token each, one of them has finished.
        dict(name="plan_8_chats", op="plan", requests=8, page_rows=16, lo=200, hi=4000, prompts=0, finished=1, dropped=0,
             longest=0, lengths=11),
        # A busy server's step: decoding requests, new prompts, finished ones, and drafts that were turned down.
        dict(name="plan_256_mixed", op="plan", requests=256, page_rows=32, lo=64, hi=16384, prompts=24, finished=9,
             dropped=31, longest=2048, lengths=23),
        # One decode step of a single user at 4k, the benchmarked head shape: latency counts.
        dict(name="decode_1_at_4097", op="decode", heads="llama_1b", kv="f32", batch=1, empty=0, page_rows=16, lo=4097,
             hi=4097, lengths=1),
        # Eight chats of 200 to 4000 positions, pages of 16 rows.
        dict(name="decode_8_chats", op="decode", heads="llama_1b", kv="f32", batch=8, empty=0, page_rows=16, lo=200,
             hi=4000, lengths=77),
        # A full server: 64 sequences of 1k to 32k positions over 16-bit pages.
        dict(name="decode_64_ragged_bf16", op="decode", heads="qwen3_8b", kv="bf16", batch=64, empty=0, page_rows=64,
             lo=1024, hi=32768, lengths=4001),
        # A batch padded to a fixed number of rows: seven query heads per kv head, biases, pages of an odd size.
        dict(name="decode_33_padded_bf16", op="decode", heads="gqa_28x4", kv="bf16", batch=33, empty=7, page_rows=24,
             lo=1, hi=9001, lengths=5),
        # Five long documents, sixteen query heads per kv head, fp32 rows.
        dict(name="decode_5_documents", op="decode", heads="mqa_32x2", kv="f32", batch=5, empty=0, page_rows=128,
             lo=4000, hi=24000, lengths=31),
        # A prompt of 8192 tokens, computed on a contiguous cache, moves into its pages.
        dict(name="scatter_8192_bf16", op="scatter", heads="qwen3_8b", kv="bf16", rows=8192, ctx=0, page_rows=64),
        # The next turn of a chat: its 1900 positions come back for the few-row kernels.
        dict(name="gather_1900", op="gather", heads="llama_1b", kv="f32", rows=1900, ctx=0, page_rows=16),
        # The key projection of one token of the 1B shape: the smallest product.
        dict(name="q4_1x2048x512", op="q4", rows=1, K=2048, N=512, group=32),
        # The output projection to a vocabulary of 128256, one token.
        dict(name="q4_1x2048x128256", op="q4", rows=1, K=2048, N=128256, group=64),
        # A gate projection for a batch of 33 requests, an odd width.
        dict(name="q4_33x2048x8200", op="q4", rows=33, K=2048, N=8200, group=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "plan", "decode", "decode", "decode", "scatter", "gather", "q4", "q4", "q4"])
    page_rows = rng.choice([8, 16, 16, 24, 32, 64, 100, 128, 256])
    if op == "plan":
        n = _log(rng, 1, 2000)
        lo = _log(rng, 1, 2000)
        prompts = rng.randint(0, n // 3)
        return dict(op=op, requests=n, page_rows=page_rows, lo=lo, hi=lo * rng.randint(1, 16), prompts=prompts,
                    finished=rng.randint(0, n // 4), dropped=rng.randint(0, n // 4),
                    longest=min(_log(rng, 1, 8192), max(1, 65536 // max(1, prompts))), lengths=rng.randint(1, 1 << 20))
    heads = rng.choice(sorted(HEADS))
    kv = rng.choice(["f32", "bf16"])
    if op == "decode":
        batch = _log(rng, 1, 100)
        most = min(32768, (250000 if kv == "f32" else 500000) // batch)
        lo = min(_log(rng, 1, 8000), most)
        hi = min(lo * rng.randint(1, 12), most)
        return dict(op=op, heads=heads, kv=kv, batch=batch, empty=rng.choice([0, 0, rng.randint(0, batch // 2)]),
                    page_rows=page_rows, lo=lo, hi=hi, lengths=rng.randint(1, 1 << 20))
    if op in ("scatter", "gather"):
        return dict(op=op, heads=heads, kv="bf16" if op == "scatter" and kv == "bf16" else "f32", rows=_log(rng, 1, 12000),
                    ctx=rng.choice([0, rng.randint(1, 500)]) if op == "scatter" else 0, page_rows=page_rows)
    K = _log(rng, 64, 12000)
    return dict(op=op, rows=rng.choice([1, 1, 2, 3, _log(rng, 1, 64)]), K=rng.choice([K, 64 * (1 + K // 64)]),
                N=_log(rng, 16, 60000), group=rng.choice([32, 64, 128]))


# ---- inputs ----

class Owned:
    """Library objects of one state, given back, newest first, when neither the state nor a tensor over their memory is
    left."""

    def __init__(self):
        self.objects = []

    def __del__(self):
        while self.objects:
            self.objects.pop().close()


class State:
    """What the program holds."""

    def __init__(self):
        self.owned = Owned()

    def keep(self, obj):
        self.owned.objects.append(obj)
        return obj


_ctx = None


def _context():
    """A program keeps one context for its device."""
    global _ctx
    if _ctx is None:
        import shainet_b200
        _ctx = shainet_b200.AttnContext(0)
    return _ctx


def _ceil(a, b):
    return -(-a // b)


def _requests(case):
    """(lengths, deltas) of a plan's requests: what the scheduler decided."""
    r = random.Random(case["lengths"])
    lens = [_log(r, case["lo"], case["hi"]) for _ in range(case["requests"])]
    delta = [1] * len(lens)
    order = list(range(len(lens)))
    r.shuffle(order)
    for i in order[:case["prompts"]]:
        lens[i], delta[i] = 0, _log(r, 1, case["longest"])
    order = order[case["prompts"]:]
    for i in order[:case["finished"]]:
        delta[i] = -lens[i]
    for i in order[case["finished"]:case["finished"] + case["dropped"]]:
        delta[i] = -r.randint(0, min(8, lens[i]))
    return lens, delta


def _lengths(case):
    """Positions of a decode batch, the new token's included; 0 is a padded row."""
    r = random.Random(case["lengths"])
    lens = [_log(r, case["lo"], case["hi"]) for _ in range(case["batch"])]
    for i in r.sample(range(len(lens)), case["empty"]):
        lens[i] = 0
    return lens


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    """The tensors of a case, on the GPU."""
    gen = torch.Generator("cuda").manual_seed(seed)
    pages_of = lambda n: torch.randperm(n, generator=gen, device="cuda").to(torch.int32)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    st = State()
    st.op = op = case["op"]
    if op == "plan":
        lens, delta = _requests(case)
        P = st.page_rows = case["page_rows"]
        st.width = _ceil(max(n + max(d, 0) for n, d in zip(lens, delta)), P) + 3
        held = [_ceil(n, P) for n in lens]
        need = sum(max(0, _ceil(n + d, P) - h) for n, d, h in zip(lens, delta, held))
        spare = need + 5 + sum(held) // 8
        st.num_pages = sum(held) + spare
        order = pages_of(st.num_pages)
        st.lens, st.delta, st.count = _ints(lens), _ints(delta), _ints([spare])
        held_t = _ints(held).long()
        at = torch.cumsum(held_t, 0) - held_t
        col = torch.arange(st.width, device="cuda")
        cell = (at[:, None] + col).clamp(max=st.num_pages - 1)
        st.table = torch.where(col < held_t[:, None], order[cell], -1).to(torch.int32).contiguous()
        st.free = torch.full((st.num_pages,), -1, dtype=torch.int32, device="cuda")
        st.free[:spare] = order[sum(held):]
        total = sum(max(d, 0) for d in delta)
        st.tokens = _ceil(total + 1, 64) * 64       # the slot array of a captured step has a fixed size
        return st
    if op == "q4":
        M, K, N, g = (case[k] for k in ("rows", "K", "N", "group"))
        st.rows, st.K, st.N, st.group = M, K, N, g
        st.packed = torch.randint(0, 256, (N, _ceil(K, 2)), generator=gen, device="cuda", dtype=torch.uint8)
        st.scales = (0.02 / 4.6) * (0.6 + 0.8 * torch.rand(N, _ceil(K, g), generator=gen, device="cuda"))
        st.x = normal(M, K)
        return st
    H, KV, hd, theta, norm, bias = HEADS[case["heads"]]
    P = st.page_rows = case["page_rows"]
    st.heads, st.kv = case["heads"], case["kv"]
    dt = torch.float32 if st.kv == "f32" else torch.bfloat16
    st.inv_freq = torch.tensor([1.0 / theta ** (2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64).to(torch.float32).cuda()
    st.norms = (1.0 + 0.02 * normal(hd), 1.0 + 0.02 * normal(hd)) if norm else None
    st.bias = (0.1 * normal(H * hd), 0.1 * normal(KV * hd), 0.1 * normal(KV * hd)) if bias else None
    if op == "decode":
        lens = _lengths(case)
        st.width = _ceil(max(max(lens), 1), P) + 2
        held = [_ceil(n, P) for n in lens]
        st.num_pages = sum(held) + 3
        st.lens = _ints(lens)
        held_t = _ints(held).long()
        at = torch.cumsum(held_t, 0) - held_t
        col = torch.arange(st.width, device="cuda")
        cell = (at[:, None] + col).clamp(max=st.num_pages - 1)
        st.table = torch.where(col < held_t[:, None], pages_of(st.num_pages)[cell], -1).to(torch.int32).contiguous()
        B = len(lens)
        st.q, st.k, st.v = normal(B, H * hd), normal(B, KV * hd), normal(B, KV * hd)
        st.scale = 1.0 / math.sqrt(hd)
    else:
        st.rows, st.ctx = case["rows"], case["ctx"]
        n = st.rows + st.ctx
        st.num_pages = _ceil(n, P) + 3
        st.width = _ceil(n, P)
        st.table = pages_of(st.num_pages)[:st.width].contiguous()
        pos = torch.arange(st.ctx, n, device="cuda")
        st.slots = (st.table[pos // P].long() * P + pos % P).to(torch.int32)
        st.ck, st.cv = (normal(KV, n, hd).to(dt) for _ in range(2))
    st.kp, st.vp = (torch.empty(st.num_pages, KV, P, hd, dtype=dt, device="cuda").normal_(generator=gen) for _ in range(2))
    return st


class _DeviceArray:
    """fp32 device memory of the library, for torch, whose tensor keeps this object and with it the memory's owner."""

    def __init__(self, ptr, shape, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<f4", "data": (ptr, False), "strides": None, "version": 3}


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        import shainet_b200 as S
        ctx = _context()
        torch.cuda.synchronize()    # the library's set-up calls work on a stream of their own
        st.stream = torch.cuda.current_stream().cuda_stream
        if st.op == "plan":
            st.lens_out, st.count_out, st.status = torch.empty_like(st.lens), torch.empty_like(st.count), _ints([0, 0])
            st.first = _ints([0] * (len(st.lens) + 1))
            st.slots = torch.empty(st.tokens, dtype=torch.int32, device="cuda")
        elif st.op == "q4":
            st.w = st.keep(S.Q4Weight.from_device(ctx, st.packed.data_ptr(), st.scales.data_ptr(), st.K, st.N, st.group))
            st.y = torch.empty(st.rows, st.N, device="cuda")
        else:
            H, KV, hd, theta = HEADS[st.heads][:4]
            kw = {}
            if st.norms:
                kw.update(q_norm=st.norms[0].cpu().numpy(), k_norm=st.norms[1].cpu().numpy())
            if st.bias:
                kw.update(zip(("b_q", "b_k", "b_v"), (b.cpu().numpy() for b in st.bias)))
            st.attn = st.keep(S.LlamaAttention(ctx, H, KV, hd, theta, EPS, kv_format=st.kv, **kw))
            st.paged = st.keep(S.PagedAttention(ctx, H, KV, hd, st.page_rows, st.kv))
            if st.op == "decode":
                st.out = torch.empty_like(st.q)
            elif st.op == "scatter":
                st.attn.cache.import_(st.ck.float().cpu().numpy(), st.cv.float().cpu().numpy())
            else:
                st.attn.cache.reserve(st.rows)
                shape = (KV, st.attn.cache.capacity, hd)
                st.got = [torch.as_tensor(_DeviceArray(p, shape, st.owned), device="cuda")[:, :st.rows]
                          for p in st.attn.cache.device_ptrs()]
    torch.cuda.synchronize()
    return st


# ---- one pass ----

def run(st):
    if own:
        return _run_own(st)
    return {"plan": _plan, "decode": _decode, "scatter": _scatter, "gather": _gather, "q4": _q4}[st.op](st)


def _run_own(st):
    import shainet_b200 as S
    if st.op == "plan":
        S.plan_pages_dev(_context(), len(st.lens), st.lens.data_ptr(), st.delta.data_ptr(), st.table.data_ptr(), st.width,
                         st.page_rows, st.free.data_ptr(), st.num_pages, st.count.data_ptr(), st.lens_out.data_ptr(),
                         st.count_out.data_ptr(), st.first.data_ptr(), st.slots.data_ptr(), st.tokens,
                         st.status.data_ptr(), stream=st.stream)
        return {"lens": st.lens_out, "count": st.count_out, "table": st.table, "free": st.free, "first": st.first,
                "slots": st.slots, "status": st.status}
    if st.op == "q4":
        st.w.gemv_dev(st.x.data_ptr(), st.y.data_ptr(), st.rows, stream=st.stream)
        return st.y
    if st.op == "decode":
        st.paged.decode_dev(st.attn, st.kp.data_ptr(), st.vp.data_ptr(), st.num_pages, st.q.data_ptr(), st.k.data_ptr(),
                            st.v.data_ptr(), st.out.data_ptr(), st.table.data_ptr(), st.width, st.lens.data_ptr(),
                            len(st.lens), st.scale, stream=st.stream)
        return {"out": st.out, "k": st.kp, "v": st.vp}
    if st.op == "scatter":
        st.paged.scatter_dev(st.attn, st.kp.data_ptr(), st.vp.data_ptr(), st.num_pages, st.slots.data_ptr(), st.ctx,
                             st.rows, stream=st.stream)
        return {"k": st.kp, "v": st.vp}
    st.paged.gather_dev(st.attn, st.kp.data_ptr(), st.vp.data_ptr(), st.num_pages, st.table.data_ptr(), st.rows,
                        stream=st.stream)
    return st.got


def _plan(st):
    P, W, NP = st.page_rows, st.width, st.num_pages
    lens, delta, free, table = st.lens.long(), st.delta.long(), st.free, st.table
    before, after = (lens + P - 1) // P, (lens + delta + P - 1) // P
    new, grow, shrink = delta.clamp(min=0), (after - before).clamp(min=0), (before - after).clamp(min=0)
    total = torch.cumsum(torch.stack([new, grow, shrink]), 1)
    new_end, grow_end, shrink_end = total
    f, r, g = st.count.long(), shrink_end[-1], grow_end[-1]
    # freed pages go on top of the stack: entry f + k is the k-th of them
    k = torch.arange(NP, device="cuda") - f
    row = torch.searchsorted(shrink_end, k, right=True).clamp(max=len(lens) - 1)
    page = table[row, (after[row] + k - (shrink_end - shrink)[row]).clamp(0, W - 1)]
    stack = torch.where((k >= 0) & (k < r), page, free)
    # the i-th page that a request grows by is the i-th from the top
    col = torch.arange(W, device="cuda")
    i = (grow_end - grow)[:, None] + col - before[:, None]
    grown = (col >= before[:, None]) & (col < after[:, None])
    cells = torch.where(grown, stack[(f + r - 1 - i).clamp(0, NP - 1)], table)
    t = torch.arange(st.tokens, device="cuda")
    row = torch.searchsorted(new_end, t, right=True).clamp(max=len(lens) - 1)
    pos = lens[row] + t - (new_end - new)[row]
    slots = torch.where(t < new_end[-1], cells[row, (pos // P).clamp(0, W - 1)] * P + pos % P, -1)
    whole = lambda x: x.to(torch.int32)
    return {"lens": whole(lens + delta), "count": whole(f + r - g), "table": cells, "free": stack,
            "first": whole(torch.cat([torch.zeros_like(new_end[:1]), new_end])), "slots": whole(slots),
            "status": torch.zeros(2, dtype=torch.int32, device="cuda")}


def _rotated(st, x, heads, norm, cos, sin):
    """[B, heads, hd] of projected rows, biased already: per-head norm and rotation, pairs (i, i + hd/2)."""
    x = x.view(len(x), heads, -1)
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _decode(st):
    H, KV, hd = HEADS[st.heads][:3]
    P, B = st.page_rows, len(st.lens)
    lens = st.lens.long()
    q, k, v = (x + b for x, b in zip((st.q, st.k, st.v), st.bias)) if st.bias else (st.q, st.k, st.v)
    last = (lens - 1).clamp(min=0)
    # the angle is the fp32 product of position and frequency, as in every cache of the package; its sine is taken in 64 bits
    angle = (last.float()[:, None] * st.inv_freq).double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    qn, kn = st.norms or (None, None)
    q, k = _rotated(st, q, H, qn, cos, sin), _rotated(st, k, KV, kn, cos, sin)
    live = torch.nonzero(lens > 0)[:, 0]
    page = st.table[live, last[live] // P].long()
    st.kp[page, :, last[live] % P] = k[live].to(st.kp.dtype)
    st.vp[page, :, last[live] % P] = v.view(B, KV, hd)[live].to(st.vp.dtype)
    cells = st.table.long().clamp(min=0)
    rows = lambda pages: pages[cells].transpose(1, 2).reshape(B, KV, st.width * P, hd).float()
    seen = (torch.arange(st.width * P, device="cuda") < lens[:, None])[:, None, None]
    scores = torch.matmul(q.reshape(B, KV, H // KV, hd), rows(st.kp).transpose(2, 3)) * st.scale
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    # a row that sees nothing is a row of zeros; values behind the last position are not looked at
    values = rows(st.vp).masked_fill(~seen.transpose(2, 3), 0.0)
    out = torch.matmul(p, values) / p.sum(-1, keepdim=True).clamp(min=1e-38)
    return {"out": out.reshape(B, H * hd), "k": st.kp, "v": st.vp}


def _scatter(st):
    slots = st.slots.long()
    for pages, cache in ((st.kp, st.ck), (st.vp, st.cv)):
        pages[slots // st.page_rows, :, slots % st.page_rows] = cache[:, st.ctx:].transpose(0, 1)
    return {"k": st.kp, "v": st.vp}


def _gather(st):
    take = lambda pages: pages[st.table.long()].transpose(0, 1).flatten(1, 2)[:, :st.rows].contiguous()
    return [take(st.kp), take(st.vp)]


def _q4(st):
    q = torch.stack([st.packed & 15, st.packed >> 4], -1).flatten(1)[:, :st.K].float() - 8.0
    s = st.scales.repeat_interleave(st.group, 1)[:, :st.K]
    return st.x @ (q * s).T


# ---- what a pass cannot do without, and its results in 64 bits ----

def work(case):
    op = case["op"]
    if op == "plan":
        lens, delta = _requests(case)
        P = case["page_rows"]
        total = sum(max(d, 0) for d in delta)
        moved = sum(abs(_ceil(n + d, P) - _ceil(n, P)) for n, d in zip(lens, delta))
        # lengths and deltas in, lengths and offsets out, slots, a page number read and written for each page that moves
        return {"bytes": 4 * (4 * len(lens) + _ceil(total + 1, 64) * 64 + 2 * moved), "flops": 8 * len(lens) + 4 * total}
    if op == "q4":
        M, K, N, g = (case[k] for k in ("rows", "K", "N", "group"))
        return {"bytes": N * _ceil(K, 2) + 4 * N * _ceil(K, g) + 4 * M * (K + N), "flops": 2 * M * N * K}
    H, KV, hd = HEADS[case["heads"]][:3]
    es = 2 if case["kv"] == "bf16" else 4
    if op == "decode":
        n = sum(_lengths(case))
        live = sum(1 for x in _lengths(case) if x)
        return {"bytes": 2 * n * KV * hd * es + live * hd * 4 * (2 * H + 2 * KV) + case["batch"] * 4 * (1 + n // (case["page_rows"] * case["batch"])),
                "flops": 4 * n * H * hd}
    return {"bytes": 4 * case["rows"] * KV * hd * es + 4 * case["rows"], "flops": 0}


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None
    st = _inputs(case, seed)
    if op == "q4":
        # a block of outputs at a time
        y = []
        for at in range(0, st.N, 4096):
            b = st.packed[at:at + 4096].to(torch.int64)
            w = torch.empty(len(b), 2 * b.shape[1], dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = b % 16 - 8, torch.div(b, 16, rounding_mode="floor") - 8
            group = torch.arange(st.K, device="cuda") // st.group
            y.append((w[:, :st.K] * st.scales[at:at + 4096].double()[:, group]) @ st.x.double().T)
        return torch.cat(y).T.contiguous()
    P = st.page_rows
    if op == "scatter":
        kp, vp = st.kp.double(), st.vp.double()
        for i in range(0, st.rows, 512):
            s = st.slots[i:i + 512].long()
            at = slice(st.ctx + i, st.ctx + i + len(s))
            kp[s // P, :, s % P], vp[s // P, :, s % P] = (c[:, at].double().permute(1, 0, 2) for c in (st.ck, st.cv))
        return {"k": kp, "v": vp}
    if op == "gather":
        found = []
        for pages in (st.kp, st.vp):
            found.append(torch.cat([pages[p] for p in st.table.tolist()], 1)[:, :st.rows].double())
        return found
    H, KV, hd, _, norm, bias = HEADS[st.heads]
    half, out = hd // 2, torch.zeros(len(st.lens), H, hd, dtype=torch.float64, device="cuda")
    new_k, new_v = [], []
    for b, n in enumerate(st.lens.tolist()):
        if n == 0:
            continue
        turn = (torch.tensor(float(n - 1), dtype=torch.float32, device="cuda") * st.inv_freq).double()
        turned = []
        for x, heads, which in ((st.q[b], H, 0), (st.k[b], KV, 1)):
            x = x.double() + (st.bias[which].double() if bias else 0.0)
            x = x.reshape(heads, hd)
            if norm:
                x = x / (x.pow(2).sum(1, keepdim=True) / hd + EPS).sqrt() * st.norms[which].double()
            z = torch.complex(x[:, :half], x[:, half:]) * torch.polar(torch.ones_like(turn), turn)
            turned.append(torch.cat([z.real, z.imag], 1))
        v = (st.v[b].double() + (st.bias[2].double() if bias else 0.0)).reshape(KV, hd)
        page, at = int(st.table[b, (n - 1) // P]), (n - 1) % P
        new_k.append((page, at, turned[1]))
        new_v.append((page, at, v))
        pages = st.table[b, :_ceil(n, P)].long()
        # attention sees the new row as the pages hold it
        keys, values = (torch.cat(list(x[pages].double().permute(0, 2, 1, 3)))[:n] for x in (st.kp, st.vp))
        keys[n - 1], values[n - 1] = turned[1].float().to(st.kp.dtype).double(), v.float().to(st.vp.dtype).double()
        for h in range(H):
            s = keys[:, h * KV // H] @ turned[0][h] * st.scale
            out[b, h] = torch.softmax(s, 0) @ values[:, h * KV // H]
    kp, vp = st.kp.double(), st.vp.double()
    for to, rows in ((kp, new_k), (vp, new_v)):
        for page, at, row in rows:
            to[page, :, at] = row
    return {"out": out.reshape(len(st.lens), H * hd), "k": kp, "v": vp}
