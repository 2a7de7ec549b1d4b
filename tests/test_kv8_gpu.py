"""The 8-bit paged cache on the GPU against plain 64-bit arithmetic: store, attention, page tables, and the three in a row."""

import math
import random

import pytest
import torch

from plain import kv8_plain as P

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture
def status():
    return torch.zeros(4, dtype=torch.int32, device="cuda")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def fine(status):
    torch.cuda.synchronize()
    assert status.tolist()[:1] == [0], status.tolist()


# ------------------------------------------------------------------------------------------------------------------ store
def same_codes(got, want):
    got, want = got.float().double().cpu(), want.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def check_store(status, *, n_pages, page, kv, d, dtype, calls, gap=0):
    """``calls``: (values maker, slots) one after the other into one pool."""
    from oxr_inference_b200 import ops

    pools = [torch.zeros((n_pages, page, kv, d), dtype=torch.float32, device="cuda").to(E4M3) for _ in range(2)]
    scales = [torch.zeros((n_pages, kv), device="cuda") for _ in range(2)]
    want = [(p.float().double().cpu(), s.double().cpu()) for p, s in zip(pools, scales)]
    for make, slots in calls:
        wide = [make(len(slots), kv * d + gap).to("cuda", dtype) for _ in range(2)]
        x = [w[:, :kv * d].unflatten(1, (kv, d)) for w in wide]
        ops.store_kv8(*x, ints(slots), *pools, *scales, status)
        fine(status)
        for i in range(2):
            want[i] = P.store(x[i].cpu(), slots, *want[i])
            assert torch.equal(scales[i].double().cpu(), want[i][1])
            same_codes(pools[i], want[i][0])


def normal(seed, factor=1.0):
    gen = torch.Generator().manual_seed(seed)
    return lambda n, w: torch.randn((n, w), generator=gen) * factor


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,kv,d", [(16, 8, 128), (1, 1, 16), (24, 3, 80), (256, 2, 48), (7, 5, 256), (16, 1, 112)])
def test_store_grows_scales(status, dtype, page, kv, d):
    """Portions, then single tokens that force the scale up by one step and by many, then ones that do not."""
    rng = random.Random(page * d)
    pages = rng.sample(range(9), 3)
    order = [p * page + o for p in pages for o in range(page)]
    a, b = len(order) // 3, len(order) // 3 + 1
    calls = [(normal(1), order[:a]), (normal(2, 3.0), order[a:b]), (normal(3, 1e4), order[b:b + 1]), (normal(4, 1e-3), order[b + 1:])]
    check_store(status, n_pages=9, page=page, kv=kv, d=d, dtype=dtype, calls=[c for c in calls if c[1]], gap=16)


def test_store_any_order_and_one_slot_twice(status):
    rng = random.Random(3)
    slots = rng.sample(range(20 * 16), 150)
    slots[7] = slots[90]
    slots[8] = slots[7]
    slots[40] = slots[41] = -1
    slots[0] = -5
    check_store(status, n_pages=20, page=16, kv=2, d=64, dtype=torch.bfloat16, calls=[(normal(5), slots), (normal(6, 9.0), slots[::-1])])


def test_store_many_tokens(status):
    """More than a thousand: one block per page for all heads."""
    rng = random.Random(4)
    slots = [p * 16 + o for p in rng.sample(range(120), 90) for o in range(16)]
    slots = slots[5:1300] + [-1] * 11
    check_store(status, n_pages=120, page=16, kv=3, d=32, dtype=torch.bfloat16, calls=[(normal(7), slots)])


def test_store_extremes(status):
    """Zeros alone, the largest and smallest magnitudes, infinities and NaN; then ordinary numbers on the same page."""
    def odd(n, w):
        x = torch.zeros((n, w))
        x[1] = 1e-30
        x[2] = 3e38
        x[3, 0], x[3, 1], x[3, 2] = math.inf, -math.inf, math.nan
        x[4] = -1e-44
        return x

    check_store(status, n_pages=6, page=2, kv=1, d=16, dtype=torch.float32,
                calls=[(odd, [0, 2, 4, 6, 8]), (normal(8), [1, 3, 5, 7, 9]), (lambda n, w: torch.zeros((n, w)), [10, 11])])


def test_store_powers_at_the_border(status):
    """Magnitudes of exactly 448 2^e, and the next ones above."""
    def border(n, w):
        x = torch.zeros((n, w))
        for i in range(n):
            x[i, 0] = 448.0 * 2.0 ** (i - 10) * (1 if i % 2 == 0 else 1 + 2.0 ** -20)
        return x

    check_store(status, n_pages=12, page=1, kv=1, d=16, dtype=torch.float32, calls=[(border, list(range(12)))])


def test_store_refuses_a_slot_outside_and_leaves_the_rest(status):
    from oxr_inference_b200 import ops

    pools = [torch.full((4, 16, 1, 16), 1.0, device="cuda").to(E4M3) for _ in range(2)]
    scales = [torch.ones((4, 1), device="cuda") for _ in range(2)]
    x = torch.ones((2, 1, 16), device="cuda")
    ops.store_kv8(x, x, ints([64, 3]), *pools, *scales, status)
    torch.cuda.synchronize()
    assert status.tolist()[0] == 2
    assert all(bool((p.float() == 1).all()) for p in pools)   # slot 3 holds 1 at scale 1 now as before


# ------------------------------------------------------------------------------------------------------------------ attention
class Batch:
    def __init__(self, q_lens, ctx_lens, *, heads, kv, d, page, dtype, seed=0, spare=2, peak=2.0):
        self.q_lens, self.ctx_lens, self.heads, self.kv, self.d, self.page, self.dtype = q_lens, ctx_lens, heads, kv, d, page, dtype
        gen = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        need = [-(-max(c, 0) // page) for c in ctx_lens]
        pages = sum(need) + spare
        order = rng.sample(range(pages), pages)
        self.tables, at = [], 0
        for n in need:
            self.tables.append(order[at:at + n])
            at += n
        width = max(need + [1])
        self.table = ints([t + [-1] * (width - len(t)) for t in self.tables])
        code = torch.randn((2, pages, page, kv, d), generator=gen) * 80
        self.k, self.v = code[0].to(E4M3).cuda(), code[1].to(E4M3).cuda()
        self.ks = torch.exp2(torch.randint(-8, -4, (pages, kv), generator=gen).float()).cuda()
        self.vs = torch.exp2(torch.randint(-9, 3, (pages, kv), generator=gen).float()).cuda()
        self.q = (torch.randn((sum(q_lens), heads, d), generator=gen) * peak / 4).to("cuda", dtype)
        cu = [0]
        for x in q_lens:
            cu.append(cu[-1] + x)
        self.cu_q, self.ctx = ints(cu), ints(ctx_lens)
        self.scale = d ** -0.5

    def run(self, status, *, window=0, out=None, q=None, **kw):
        from oxr_inference_b200 import ops

        how = dict(max_q_len=max(self.q_lens + [1]), kv_len_bound=max(self.ctx_lens + [1]))
        how.update(kw)
        return ops.paged_attention_kv8(self.q if q is None else q, self.k, self.v, self.ks, self.vs, cu_q=self.cu_q, ctx_lens=self.ctx, block_table=self.table,
                                       scale=self.scale, window=window, status=status, out=out, **how)

    def check(self, status, *, window=0, **kw):
        got = self.run(status, window=window, **kw)
        fine(status)
        assert got.dtype == self.dtype
        want, spread, size = P.attention(self.q, self.k.float(), self.v.float(), self.ks, self.vs, self.q_lens, self.ctx_lens, self.tables, self.scale, window)
        tol = P.tolerance(want, spread, size, self.dtype, self.d, max(self.ctx_lens + [1]))
        off = (got.double().cpu() - want).abs()
        assert bool((off <= tol).all()), float((off / tol).max())


DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,d,page", [(32, 8, 128, 16), (4, 4, 16, 8), (6, 2, 48, 16), (12, 4, 80, 24), (16, 1, 64, 1), (40, 2, 128, 64), (3, 1, 112, 7), (5, 1, 256, 16), (8, 2, 32, 300)])
def test_attention_single_tokens(status, dtype, heads, kv, d, page):
    Batch([1] * 5, [1, 31, 32, 257, 64], heads=heads, kv=kv, d=d, page=page, dtype=dtype).check(status)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,d,page", [(8, 2, 128, 16), (4, 4, 64, 32), (6, 1, 80, 24), (4, 1, 256, 16)])
@pytest.mark.parametrize("window", [0, 1, 33])
def test_attention_mixed_lengths(status, dtype, heads, kv, d, page, window):
    """Requests without a token, with one, with a few and with many; contexts that end inside a page and a block of keys."""
    Batch([0, 1, 7, 3, 0, 8, 41, 1, 0], [40, 77, 7, 130, 0, 33, 90, 1, 5], heads=heads, kv=kv, d=d, page=page, dtype=dtype).check(status, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_few_requests_share_their_keys(status, dtype):
    """One long request: its keys are cut between the blocks of a cluster."""
    Batch([1], [3001], heads=4, kv=1, d=64, page=16, dtype=dtype).check(status)
    Batch([2, 1], [1500, 3], heads=8, kv=2, d=128, page=16, dtype=dtype, seed=1).check(status)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bound", [1, 100000])
def test_attention_a_wrong_length_bound_changes_nothing_but_the_cut(status, dtype, bound):
    Batch([1, 2], [700, 90], heads=4, kv=2, d=64, page=16, dtype=dtype).check(status, kv_len_bound=bound)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_rows_that_see_nothing_are_zero(status, dtype):
    """Contexts shorter than the new tokens: the first ones stand before the sequence."""
    b = Batch([5, 1, 3], [2, 0, 3], heads=4, kv=2, d=32, page=16, dtype=dtype)
    b.check(status)
    got = b.run(status)
    assert bool((got[:3] == 0).all()) and bool((got[5] == 0).all()) and bool((got[3] != 0).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [0, 20])
def test_attention_what_is_hidden_may_hold_anything(status, dtype, window):
    """NaN codes and NaN, infinite and negative scales behind the context, before the window and at later tokens of the same request."""
    b = Batch([3, 1, 6], [50, 70, 45], heads=4, kv=2, d=64, page=16, dtype=dtype, seed=2)
    for r, ctx in enumerate(b.ctx_lens):   # behind the context, on its last page and on pages that no table names
        for o in range(ctx % 16, 16):
            b.k.view(torch.uint8)[b.tables[r][-1], o] = 0x7F
            b.v.view(torch.uint8)[b.tables[r][-1], o] = 0xFF
    if window:   # a whole page before every window of request 1
        b.k.view(torch.uint8)[b.tables[1][0]] = 0x7F
        b.v.view(torch.uint8)[b.tables[1][1]] = 0x7F
        b.ks[b.tables[1][0]] = math.nan
        b.vs[b.tables[1][1]] = math.inf
    b.check(status, window=window)
    # the last token's own value is NaN in one entry: the tokens before it must not notice
    last = b.ctx_lens[2] - 1
    want = b.run(status, window=window)
    b.v.view(torch.uint8)[b.tables[2][last // 16], last % 16, 0, 5] = 0x7F
    got = b.run(status, window=window)
    fine(status)
    assert torch.equal(got[:9], want[:9])
    assert bool(torch.isnan(got[9, :2, 5]).all())
    clean = torch.ones(64, dtype=torch.bool)
    clean[5] = False
    assert torch.equal(got[9][:, clean], want[9][:, clean]) and torch.equal(got[9, 2:], want[9, 2:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_nan_reaches_its_rows_alone(status, dtype):
    b = Batch([1, 1], [40, 40], heads=4, kv=2, d=64, page=16, dtype=dtype)
    want = b.run(status)
    b.q[0, 1, 3] = math.nan
    got = b.run(status)
    fine(status)
    assert bool(torch.isnan(got[0, 1]).all())
    got[0, 1] = want[0, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("exponents", [(-118, -118), (100, 100), (-60, 20), (0, 0)])
def test_attention_scales_of_any_size(status, dtype, exponents):
    """Pages whose value scales are all tiny, all large, far apart, or zero; key scales that are no power of two."""
    b = Batch([1, 3], [90, 75], heads=4, kv=2, d=64, page=16, dtype=dtype, seed=3)
    gen = torch.Generator().manual_seed(1)
    e = torch.randint(exponents[0], exponents[1] + 1, b.vs.shape, generator=gen).float()
    b.vs = torch.ldexp(torch.ones_like(e), e.int()).cuda()
    if exponents == (0, 0):
        b.vs[b.tables[0][0]] = 0
        b.vs[b.tables[1][-1]] = 0
    b.ks *= 1.37
    b.check(status)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("factor", [1e-30, 1e-3, 40.0])
def test_attention_queries_of_any_size(status, dtype, factor):
    b = Batch([1, 2], [300, 65], heads=8, kv=2, d=128, page=16, dtype=dtype, seed=4)
    b.q = (b.q.float() * factor).to(dtype)
    b.check(status)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_attention_scale_of_any_sign(status, dtype, scale):
    b = Batch([1, 9], [300, 65], heads=8, kv=2, d=64, page=16, dtype=dtype, seed=5)
    b.scale = scale
    b.check(status)


def test_attention_one_large_weight_and_a_long_tail(status):
    """A first key that takes most of the weight and thousands of keys with 2^-14 of it each: together they count."""
    n = 4000
    b = Batch([1], [n], heads=1, kv=1, d=16, page=16, dtype=torch.bfloat16)
    k = torch.zeros((b.k.shape[0], 16, 1, 16))
    k[b.tables[0][0], 0] = 1
    b.k, b.v = k.to(E4M3).cuda(), torch.ones_like(k).to(E4M3).cuda()
    b.v[b.tables[0][0], 0] = -1
    b.ks.fill_(1), b.vs.fill_(1)
    b.q.fill_(1)
    b.scale = 14 * math.log(2) / 16
    b.check(status)


def test_attention_strides_out_and_rows_behind(status):
    """Queries that are columns of a wider product, pools that interleave keys and values, a given output with rows behind the last sequence."""
    for dtype in DTYPES:
        b = Batch([1, 4, 2], [60, 35, 90], heads=4, kv=2, d=64, page=16, dtype=dtype, seed=6)
        want = b.run(status)
        both = torch.stack([b.k.view(torch.uint8), b.v.view(torch.uint8)], 1).view(E4M3)
        b.k, b.v = both[:, 0], both[:, 1]
        wide = torch.full((9, 6 * 64), math.nan, dtype=dtype, device="cuda")
        wide[:7, 64:64 * 5] = b.q.flatten(1)
        q = wide[:, 64:64 * 5].unflatten(1, (4, 64))
        out = torch.full((9, 4, 64), 7.0, dtype=dtype, device="cuda")
        got = b.run(status, q=q, out=out)
        fine(status)
        assert got is out and torch.equal(got[:7], want) and bool((got[7:] == 7).all())


def test_attention_bad_pages_and_lengths_are_reported(status):
    b = Batch([1, 1], [40, 40], heads=4, kv=2, d=64, page=16, dtype=torch.bfloat16)
    want = b.run(status)
    for bad in (-1, b.k.shape[0], 1 << 30):
        table = b.table.clone()
        b.table[1, 1] = bad
        got = b.run(status)
        torch.cuda.synchronize()
        assert status.tolist()[0] == 4
        assert torch.equal(got[0], want[0])
        status.zero_()
        b.table = table
    b.ctx = ints([40, 49])   # longer than the table's three pages
    b.run(status)
    torch.cuda.synchronize()
    assert status.tolist()[0] == 4
    status.zero_()
    b = Batch([1, 3, 20], [40, 40, 40], heads=4, kv=2, d=64, page=16, dtype=torch.bfloat16)
    for most in (1, 2, 8):
        b.run(status, max_q_len=most)
        torch.cuda.synchronize()
        assert status.tolist()[0] == 100, most
        status.zero_()


def test_attention_bounds_beyond_all_sizes(status):
    """A window, a number of new tokens and a length that no 32-bit number holds mean none at all. (They decide how the keys are cut, and with it the order
    of the sums.)"""
    Batch([1, 4, 2], [60, 35, 90], heads=4, kv=2, d=64, page=16, dtype=torch.bfloat16).check(status, window=1 << 40, max_q_len=1 << 40, kv_len_bound=1 << 40)


def test_attention_far_pages(status):
    """Pages beyond 2^31 bytes of the pool."""
    d, kv, page = 128, 8, 64
    pages = (1 << 31) // (page * kv * d) + 3
    b = Batch([1], [60], heads=8, kv=kv, d=d, page=page, dtype=torch.bfloat16)
    want = b.run(status)
    far = pages - 2
    k, v = (torch.zeros((pages, page, kv, d), dtype=torch.uint8, device="cuda") for _ in range(2))
    k[far], v[far] = b.k.view(torch.uint8)[b.tables[0][0]], b.v.view(torch.uint8)[b.tables[0][0]]
    ks, vs = (torch.zeros((pages, kv), device="cuda") for _ in range(2))
    ks[far], vs[far] = b.ks[b.tables[0][0]], b.vs[b.tables[0][0]]
    b.k, b.v, b.ks, b.vs = k.view(E4M3), v.view(E4M3), ks, vs
    b.table = ints([[far]])
    got = b.run(status)
    fine(status)
    assert torch.equal(got, want)


def test_attention_replayed_and_on_two_streams(status):
    b = Batch([1, 1, 1], [700, 90, 33], heads=8, kv=2, d=128, page=16, dtype=torch.bfloat16)
    want = b.run(status)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            got.append(b.run(status))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.run(status)
    b.q.copy_(b.q.flip(0))
    graph.replay()
    fine(status)
    assert torch.equal(out, b.run(status))


# ------------------------------------------------------------------------------------------------------------------ page tables
def tables_case(rows, page, width, seed, *, most_new=1, fresh=0.2, idle=0.1):
    rng = random.Random(seed)
    lengths = [rng.choice([0, 1, page, page + 1, rng.randint(0, width * page // 2)]) for _ in range(rows)]
    held = [min(width, -(-n // page) + rng.choice([0, 0, 1])) for n in lengths]
    new = [0 if rng.random() < idle else rng.randint(1, most_new) for _ in range(rows)]
    anew = [int(rng.random() < fresh) for _ in range(rows)]
    pool = sum(held) + sum(-(-(q + page) // page) for q in new) + 7
    ids = rng.sample(range(pool), pool)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-7] * (width - h))
        at += h
    return lengths, held, table, (ids[at:] + [-3] * at, pool - at), new, anew


def run_tables(case, page, tokens, status, **kw):
    from oxr_inference_b200 import ops

    lengths, held, table, (stack, count), new, anew = case
    state = [ints(lengths), ints(held), ints(table).view(len(lengths), len(table[0]) if table else 4), ints(stack), ints([count])]
    step = ops.step_pages(*state, ints(new), ints(anew), page_size=page, tokens=tokens, status=status, **kw)
    torch.cuda.synchronize()
    return state, step


@pytest.mark.parametrize("rows,page,width,most_new,spare", [(1, 16, 4, 1, 0), (7, 16, 20, 1, 3), (256, 16, 40, 1, 0), (33, 8, 90, 200, 50), (5, 1, 3000, 900, 0),
                                                           (1500, 24, 12, 2, 1), (8192, 16, 3, 1, 9), (3, 4096, 2, 3000, 1)])
@pytest.mark.parametrize("advance", [False, True])
def test_tables(status, rows, page, width, most_new, spare, advance):
    case = tables_case(rows, page, width, rows + page, most_new=most_new)
    lengths, held, table, free, new, anew = case
    tokens = sum(new) + spare
    state, step = run_tables(case, page, tokens, status, advance=advance)
    fine(status)
    held2, table2, stack, count, begin, cu = P.pages(lengths, held, table, free, new, anew, page)
    after = [b + q for b, q in zip(begin, new)]
    assert state[0].tolist() == (after if advance else lengths)
    assert state[1].tolist() == held2 and state[2].tolist() == table2 and state[3].tolist() == stack and state[4].tolist() == [count]
    assert step.cu_q.tolist() == cu and step.ctx_lens.tolist() == after
    pos = [b + i for b, q in zip(begin, new) for i in range(q)]
    req = [r for r, q in enumerate(new) for _ in range(q)]
    assert step.positions.tolist() == pos + [0] * spare
    assert step.req_of_token.tolist() == req + [-1] * spare
    assert step.slots.tolist() == [table2[r][p // page] * page + p % page for r, p in zip(req, pos)] + [-1] * spare


def test_tables_asked_twice_take_nothing_more(status):
    case = tables_case(40, 16, 30, 5, most_new=30, fresh=0.0)
    state, first = run_tables(case, 16, sum(case[4]), status)
    from oxr_inference_b200 import ops

    before = [s.clone() for s in state]
    again = ops.step_pages(*state, ints(case[4]), None, page_size=16, tokens=sum(case[4]), status=status)
    fine(status)
    assert all(torch.equal(a, b) for a, b in zip(state, before)) and all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("what,code", [("pages", 6), ("row", 7), ("negative", 7), ("tokens", 8), ("stack", 6)])
@pytest.mark.parametrize("rows", [20, 2000])
def test_tables_all_or_nothing(status, what, code, rows):
    lengths, held, table, (stack, count), new, anew = tables_case(rows, 16, 12, 3, most_new=20, fresh=0.0)
    tokens = sum(new)
    if what == "pages":
        count = 1
    elif what == "row":
        new[rows // 2] += 12 * 16
        tokens = sum(new)
    elif what == "negative":
        new[rows // 2] = -1
    elif what == "tokens":
        tokens -= 1
    else:   # more is given back than the stack has room for
        anew[:] = [1] * rows
        count, stack = 5, stack[:6]
    state, step = run_tables((lengths, held, table, (stack, count), new, anew), 16, tokens, status)
    assert status.tolist()[0] == code
    assert state[0].tolist() == lengths and state[1].tolist() == held and state[2].tolist() == table and state[3].tolist() == stack and state[4].tolist() == [count]
    assert set(step.slots.tolist()) <= {-1} and set(step.req_of_token.tolist()) <= {-1}
    assert set(step.cu_q.tolist()) == {0} and set(step.ctx_lens.tolist()) == {0}


def test_tables_without_rows_or_tokens(status):
    state, step = run_tables(([], [], [], ([4, 5], 2), [], []), 16, 3, status)
    fine(status)
    assert step.cu_q.tolist() == [0] and step.slots.tolist() == [-1] * 3 and state[4].tolist() == [2]
    state, step = run_tables(([5], [1], [[0, 9]], ([4, 5, -1], 2), [0], [1]), 16, 0, status)   # a row is given up
    fine(status)
    assert state[4].tolist() == [3] and state[3].tolist() == [4, 5, 0]
    assert state[1].tolist() == [0] and step.ctx_lens.tolist() == [0]


# ------------------------------------------------------------------------------------------------------------------ in a row
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_prompt_and_its_decoding_in_a_graph(status, dtype):
    """Prompts of several requests, then decode steps replayed from one graph that holds tables, store and attention; every step's result against
    64 bits over what the cache ought to hold."""
    from oxr_inference_b200 import ops

    page, kv, heads, d, rows = 8, 2, 4, 32, 3
    prompts, steps = [13, 8, 3], 12
    gen = torch.Generator().manual_seed(9)
    pool = 40
    lengths, held, table = ints([0] * rows), ints([0] * rows), ints([[-1] * 10] * rows)
    free_list, free_count = ints(random.Random(1).sample(range(pool), pool)), ints([pool])
    k_cache, v_cache = (torch.zeros((pool, page, kv, d), dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    k_scale, v_scale = (torch.zeros((pool, kv), device="cuda") for _ in range(2))
    want = [(c.float().double().cpu(), s.double().cpu()) for c, s in ((k_cache, k_scale), (v_cache, v_scale))]

    def made(n, h):
        return (torch.randn((n, h, d), generator=gen) * torch.exp(torch.randn((n, 1, 1), generator=gen))).to("cuda", dtype)

    def layer(q, k, v, q_lens, most, tokens):
        s = ops.step_pages(lengths, held, table, free_list, free_count, q_lens, page_size=page, tokens=tokens, status=status, advance=True)
        ops.store_kv8(k, v, s.slots, k_cache, v_cache, k_scale, v_scale, status)
        return s, ops.paged_attention_kv8(q, k_cache, v_cache, k_scale, v_scale, cu_q=s.cu_q, ctx_lens=s.ctx_lens, block_table=table, scale=0.3,
                                          max_q_len=most, kv_len_bound=40, status=status)

    def check(s, o, q, k, v, new):
        fine(status)
        slots = s.slots.tolist()
        for i, x in enumerate((k, v)):
            want[i] = P.store(x.cpu(), slots, *want[i])
        same_codes(k_cache, want[0][0])
        same_codes(v_cache, want[1][0])
        tables = [r[:h] for r, h in zip(table.tolist(), held.tolist())]
        ref, spread, size = P.attention(q, want[0][0], want[1][0], want[0][1], want[1][1], new, lengths.tolist(), tables, 0.3)
        assert bool(((o.double().cpu() - ref).abs() <= P.tolerance(ref, spread, size, dtype, d, 40)).all())

    q, k, v = made(sum(prompts), heads), made(sum(prompts), kv), made(sum(prompts), kv)
    check(*layer(q, k, v, ints(prompts), max(prompts), sum(prompts)), q, k, v, prompts)
    q, k, v, ones = made(rows, heads), made(rows, kv), made(rows, kv), ints([1] * rows)
    keep = [t.clone() for t in (lengths, held, table, free_list, free_count, k_cache.view(torch.uint8), v_cache.view(torch.uint8), k_scale, v_scale)]
    layer(q, k, v, ones, 1, rows)   # libraries are loaded before the capture
    for t, was in zip((lengths, held, table, free_list, free_count, k_cache.view(torch.uint8), v_cache.view(torch.uint8), k_scale, v_scale), keep):
        t.copy_(was)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s, o = layer(q, k, v, ones, 1, rows)
    for _ in range(steps):
        for t, h in ((q, heads), (k, kv), (v, kv)):
            t.copy_(made(rows, h))
        graph.replay()
        check(s, o, q, k, v, [1] * rows)
    assert lengths.tolist() == [p + steps for p in prompts]


def test_tables_of_page_numbers_beyond_all_pools(status):
    """They do not come round to the pages below: 2^29 pages of 8 are as many slots as 32 bits count."""
    far = [1 << 28, 1 << 29, (1 << 29) + 3, (1 << 31) - 1, -2, 5]
    case = ([8] * 6, [2] * 6, [[0, f] for f in far], ([1, 2, 3], 3), [1] * 6, [0] * 6)
    state, step = run_tables(case, 8, 6, status)
    fine(status)
    assert step.slots.tolist() == [(1 << 31) - 1] * 4 + [-1, 40]
