"""Block tables and slot maps built on the device (shainet_attn_paged_plan_dev) against a plain host scheduler that keeps
Python lists: whole numbers, so everything is compared for equality, what is not in use included."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
OK, SHORT, LENGTH, TOKENS, STACK = range(5)


@pytest.fixture(scope="module")
def ctx():
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    yield c
    c.close()


def host_plan(lens, delta, table, P, free, count, tokens):
    """(status, lens, count, table, free, first, slots) of one step, by the definition."""
    R, W, NP = len(lens), table.shape[1], len(free)
    same = lambda code, detail: ([code, detail], lens, count, table, free, np.zeros(R + 1, np.int32), np.full(tokens, -1, np.int32))
    table, free = table.copy(), free.copy()
    pages = lambda n: -(-n // P)
    for r in range(R):
        if not 0 <= lens[r] <= W * P or not 0 <= int(lens[r]) + int(delta[r]) <= W * P:
            return same(LENGTH, r)
    freed = [table[r, c] for r in range(R) for c in range(pages(lens[r] + delta[r]), pages(lens[r]))]
    if count < 0 or count + len(freed) > NP:
        return same(STACK, count)
    total = sum(max(0, int(d)) for d in delta)
    if total > tokens:
        return same(TOKENS, total)
    need = sum(max(0, pages(lens[r] + delta[r]) - pages(lens[r])) for r in range(R))
    if need > count + len(freed):
        return same(SHORT, need - count - len(freed))
    before_table = table.copy()
    stack = list(free[:count]) + freed
    free[count:count + len(freed)] = freed
    slots, first = [], [0]
    for r in range(R):
        for c in range(pages(lens[r]), pages(lens[r] + delta[r])):
            table[r, c] = stack.pop()
        for p in range(lens[r], lens[r] + max(0, delta[r])):
            slots.append(table[r, p // P] * P + p % P)
        first.append(len(slots))
    assert (before_table[lens + delta < lens] == table[lens + delta < lens]).all()
    slots += [-1] * (tokens - len(slots))
    return [OK, 0], lens + delta, len(stack), table, free, np.array(first, np.int32), np.array(slots, np.int32)


def state(rng, R, W, P, NP, lens, spare):
    """A table whose requests hold distinct random pages; cells and stack entries that are not in use hold a marker."""
    order = rng.permutation(NP).astype(np.int32)
    table = np.full((R, W), -7, np.int32)
    at = 0
    for r in range(R):
        n = -(-int(lens[r]) // P)
        table[r, :n] = order[at:at + n]
        at += n
    free = np.full(NP, -9, np.int32)
    assert at + spare <= NP
    free[:spare] = order[at:at + spare]
    return table, free


def device_plan(ctx, lens, delta, table, P, free, count, tokens, in_place=False, stream=None):
    import torch
    import shainet_b200 as S
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()
    guard = 3
    tl, td, tt, tf, tc = dev(lens), dev(delta), dev(table), dev(free), dev([count])
    lo, co = (tl, tc) if in_place else (torch.full_like(tl, -5), torch.full_like(tc, -5))
    R = len(lens)
    first = torch.full((R + 1 + guard,), -5, dtype=torch.int32, device="cuda")
    slots = torch.full((tokens + guard,), -5, dtype=torch.int32, device="cuda")
    status = torch.full((2 + guard,), -5, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    S.plan_pages_dev(ctx, R, tl.data_ptr(), td.data_ptr(), tt.data_ptr(), table.shape[1], P, tf.data_ptr(), len(free), tc.data_ptr(),
                     lo.data_ptr(), co.data_ptr(), first.data_ptr(), slots.data_ptr(), tokens, status.data_ptr(), stream=stream)
    ctx.sync()
    torch.cuda.synchronize()
    get = lambda t: t.cpu().numpy()
    assert (get(first)[R + 1:] == -5).all() and (get(slots)[tokens:] == -5).all() and (get(status)[2:] == -5).all()
    return list(get(status)[:2]), get(lo), int(get(co)[0]), get(tt), get(tf), get(first)[:R + 1], get(slots)[:tokens]


def check(ctx, *args, **kw):
    want, got = host_plan(*args), device_plan(ctx, *args, **kw)
    for name, w, g in zip(("status", "lens", "count", "table", "free", "first", "slots"), want, got):
        assert np.array_equal(np.asarray(w), np.asarray(g)), name
    return want


def mixed(rng, R, P, longest):
    """Decoding, starting, finished, shortened and idle requests."""
    lens = rng.integers(0, 6 * P, R)
    kind = rng.integers(0, 6, R)
    delta = np.where(kind == 0, -lens, np.where(kind == 1, -np.minimum(lens, rng.integers(0, 2 * P, R)), np.where(kind == 2, 0, 1)))
    starts = kind == 3
    lens[starts] = 0
    delta[starts] = rng.integers(1, longest + 1, starts.sum())
    return lens.astype(np.int32), delta.astype(np.int32)


@pytest.mark.parametrize("in_place", [False, True], ids=["out", "in_place"])
@pytest.mark.parametrize("R,P,longest", [(1, 16, 40), (2, 1, 5), (7, 24, 100), (33, 16, 300), (256, 32, 700), (1000, 8, 60),
                                         (1025, 3, 9), (2500, 16, 20), (8192, 5, 3)])
def test_mixed_steps(ctx, R, P, longest, in_place):
    rng = np.random.default_rng(R * 100 + P)
    lens, delta = mixed(rng, R, P, longest)
    W = int(max(np.maximum(lens, lens + delta).max(), 1) + P - 1) // P + 2
    held, after = (lens + P - 1) // P, (lens + delta + P - 1) // P
    need = int(np.maximum(after - held, 0).sum())
    NP = int(held.sum()) + need + 4
    table, free = state(rng, R, W, P, NP, lens, need)
    total = int(np.maximum(delta, 0).sum())
    for tokens in (total, total + 37):
        assert check(ctx, lens, delta, table, P, free, need, tokens, in_place=in_place)[0] == [OK, 0]


def test_freed_pages_are_popped_in_the_same_step(ctx):
    """No free page at all: what finished and shortened requests give up is what the others grow by; then one page short."""
    rng = np.random.default_rng(5)
    P, W = 16, 12
    lens = np.array([100, 0, 33, 48, 17, 160, 5], np.int32)
    delta = np.array([-100, 120, -20, 1, 31, -81, 0], np.int32)
    table, free = state(rng, len(lens), W, P, 40, lens, 0)
    assert check(ctx, lens, delta, table, P, free, 0, 200)[0] == [OK, 0]
    delta[1] = 176     # 11 pages instead of 8
    status = check(ctx, lens, delta, table, P, free, 0, 300)[0]
    assert status[0] in (OK, SHORT)
    delta[4] = 140
    assert check(ctx, lens, delta, table, P, free, 0, 400)[0][0] == SHORT


def test_large_prompts_take_the_cluster(ctx):
    rng = np.random.default_rng(6)
    P, lens = 16, np.array([0, 31, 0, 7, 0], np.int32)
    delta = np.array([30000, 1, 8191, 25000, 0], np.int32)
    table, free = state(rng, 5, 2000, P, 5000, lens, 4800)
    for in_place in (False, True):
        assert check(ctx, lens, delta, table, P, free, 4800, 65536, in_place=in_place)[0] == [OK, 0]
    assert check(ctx, lens, delta, table, P, free, 100, 65536, in_place=True)[0][0] == SHORT


@pytest.mark.parametrize("tokens", [40, 20000], ids=["one_cta", "cluster"])
@pytest.mark.parametrize("what", ["negative_length", "long_length", "below_zero", "past_the_table", "overflow", "tokens", "count_below",
                                  "count_above", "stack_overflow", "empty"])
def test_steps_that_cannot_be_taken_change_nothing(ctx, what, tokens):
    rng = np.random.default_rng(7)
    P, W, NP = 16, 8, 60
    lens = np.array([20, 40, 0, 128, 64], np.int32)
    delta = np.array([1, -8, 10, 0, 1], np.int32)
    table, free = state(rng, 5, W, P, NP, lens, 10)
    count, want = 10, None
    if what == "negative_length": lens[2], want = -3, [LENGTH, 2]
    if what == "long_length": lens[4], want = 129, [LENGTH, 4]
    if what == "below_zero": delta[1], want = -41, [LENGTH, 1]
    if what == "past_the_table": delta[3], want = 1, [LENGTH, 3]
    if what == "overflow": lens[0], delta[0], want = 100, 2**31 - 1, [LENGTH, 0]
    if what == "tokens":
        if tokens > 40: pytest.skip("the array is large enough")
        delta[2], delta[0], want = 30, 20, [TOKENS, 51]
    if what == "count_below": count, want = -1, [STACK, -1]
    if what == "count_above": count, want = NP + 1, [STACK, NP + 1]
    if what == "stack_overflow":
        delta[1], count, want = -40, NP - 2, [STACK, NP - 2]
    if what == "empty": want = [OK, 0]
    for in_place in (False, True):
        assert check(ctx, lens, delta, table, P, free, count, tokens, in_place=in_place)[0] == want


def test_pages_outside_the_pool_have_no_slots(ctx):
    """A table cell or a free page that is not a page: its slots are -1, also where page * page_rows would wrap to a slot
    of the pool; the rest of the step is taken."""
    P, NP = 16, 6
    lens, delta = np.array([5, 20, 16, 3], np.int32), np.array([2, 1, 2, 2], np.int32)
    table, free = np.array([[1 << 28, -7], [0, 1], [2, -7], [-1, -7]], np.int32), np.array([3, 4, NP, -9, -9, -9], np.int32)
    status, _, count, tab, _, first, slots = device_plan(ctx, lens, delta, table, P, free, 3, 12)
    assert status == [OK, 0] and count == 2 and list(first) == [0, 2, 3, 5, 7] and tab[2, 1] == NP
    assert list(slots) == [-1, -1, 20, -1, -1, -1, -1] + [-1] * 5


def test_the_longest_slot_map(ctx):
    """2^31 - 1 places for slots: the last step of the loop that fills them passes 2^31."""
    import torch
    import shainet_b200 as S
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    tokens = 2**31 - 1
    dev = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    lens, delta, table, count, first, status = dev(15), dev(3), dev(4, -7), dev(2), dev(-5, -5), dev(-5, -5)
    slots = torch.full((tokens + 8192,), -5, dtype=torch.int32, device="cuda")      # no guard before it: the front is checked too
    for page_rows, left, pages in ((16, 1, 3), (17, 1, 3), (16, 1, 10)):     # pages 4, 8 and 9: outside a pool of three
        free = dev(9, 8, *[-9] * (pages - 2))
        lens.fill_(page_rows - 1)
        count.fill_(2)
        slots.fill_(-5)
        torch.cuda.synchronize()
        S.plan_pages_dev(ctx, 1, lens.data_ptr(), delta.data_ptr(), table.data_ptr(), 2, page_rows, free.data_ptr(), pages, count.data_ptr(),
                         lens.data_ptr(), count.data_ptr(), first.data_ptr(), slots.data_ptr(), tokens, status.data_ptr())
        ctx.sync()
        assert status.tolist() == [OK, 0] and lens.item() == page_rows + 2 and count.item() == left and table.tolist() == [4, 8]
        assert slots[:3].tolist() == ([4 * page_rows + page_rows - 1, 8 * page_rows, 8 * page_rows + 1] if pages > 8 else [-1, -1, -1])
        assert bool((slots[3:tokens] == -1).all()) and bool((slots[tokens:] == -5).all())


def test_no_requests_and_no_tokens(ctx):
    free = np.arange(4, dtype=np.int32)
    empty = np.zeros(0, np.int32)
    check(ctx, empty, empty, np.zeros((0, 3), np.int32), 16, free, 4, 5)
    lens, delta = np.array([17], np.int32), np.array([-17], np.int32)
    check(ctx, lens, delta, np.array([[2, 3, -7]], np.int32), 16, np.array([0, 1, -9, -9], np.int32), 2, 0)


def test_captured_step_advances_its_own_state(ctx):
    """A serving loop as one graph: lens and free_count in place, replayed; the host scheduler runs beside it."""
    import torch
    import shainet_b200 as S
    rng = np.random.default_rng(8)
    P, W, NP, R, tokens = 4, 40, 400, 9, 16
    lens = rng.integers(1, 60, R).astype(np.int32)
    delta = np.ones(R, np.int32)
    table, free = state(rng, R, W, P, NP, lens, 200)
    count = 200
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()
    tl, td, tt, tf, tc = dev(lens), dev(delta), dev(table), dev(free), dev([count])
    first, slots, status = dev(np.zeros(R + 1)), dev(np.zeros(tokens)), dev([9, 9])
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        S.plan_pages_dev(ctx, R, tl.data_ptr(), td.data_ptr(), tt.data_ptr(), W, P, tf.data_ptr(), NP, tc.data_ptr(), tl.data_ptr(),
                         tc.data_ptr(), first.data_ptr(), slots.data_ptr(), tokens, status.data_ptr(), stream=stream.cuda_stream)
    for step in range(30):
        delta = rng.integers(-3, 2, R).astype(np.int32)
        delta = np.maximum(delta, -lens)
        if step == 20: delta[4] = -lens[4]
        td.copy_(dev(delta))
        graph.replay()
        torch.cuda.synchronize()
        want = host_plan(lens, delta, table, P, free, count, tokens)
        got = [list(status.cpu().numpy()), tl.cpu().numpy(), int(tc[0]), tt.cpu().numpy(), tf.cpu().numpy(), first.cpu().numpy(),
               slots.cpu().numpy()]
        for w, g in zip(want, got):
            assert np.array_equal(np.asarray(w), np.asarray(g)), step
        _, lens, count, table, free = want[:5]
