"""Attention over 8-bit pages whose scales are far apart: in a block of keys, between blocks, in the sight of a row or out of it."""

import math
import random

import pytest
import torch

from oxr_inference_b200.ops import kv8
from plain import kv8_plain as P
from test_kv8_gpu import DTYPES, E4M3, Batch, fine, status  # noqa: F401

pytestmark = pytest.mark.gpu
LOWEST, HIGHEST = -118, 120      # exponents of the scales that the store makes

# (name, type of the queries, head size, new tokens of two requests, their contexts): the split-key kernel with its two sizes of tiles and both types
SPLIT = [("few", dtype, 64, [1, 3], [170, 150]) for dtype in DTYPES] + [("rows16", dtype, 128, [6, 8], [170, 150]) for dtype in DTYPES]


def sizes(case, page=16, **kw):
    _, dtype, d, q_lens, ctx_lens = case
    return Batch(q_lens, ctx_lens, heads=4, kv=2, d=d, page=page, dtype=dtype, **kw)


def powers(exponents):
    e = torch.as_tensor(exponents, dtype=torch.float32)
    return torch.ldexp(torch.ones_like(e), e.int()).cuda()


def tame(b):
    """Codes of at most 240, so that 2^120 times one is a float32 number."""
    b.v = b.v.float().clamp(-240, 240).to(E4M3)


def name_of(case):
    return f"{case[0]}-{'bf16' if case[1] == torch.bfloat16 else 'fp32'}"


@pytest.mark.parametrize("case", SPLIT, ids=name_of)
@pytest.mark.parametrize("seed", range(10))
def test_value_scales_over_all_that_the_store_makes(status, case, seed):  # noqa: F811
    b = sizes(case, seed=seed)
    tame(b)
    gen = torch.Generator().manual_seed(seed)
    low, high = ((LOWEST, HIGHEST), (-60, 20), (-12, 12), (-3, 3))[seed % 4]
    b.vs = powers(torch.randint(low, high + 1, b.vs.shape, generator=gen))
    b.check(status)


@pytest.mark.parametrize("case", SPLIT, ids=name_of)
@pytest.mark.parametrize("first,last", [(LOWEST, 12), (12, LOWEST), (5, LOWEST), (LOWEST, HIGHEST), (HIGHEST, LOWEST), (-40, 40), (40, -40)])
@pytest.mark.parametrize("cut", [1, 4, 9])
def test_two_value_scales(status, case, first, last, cut):  # noqa: F811
    """The first ``cut`` pages of each request at one scale, the others at another: inside a block of keys and between blocks."""
    b = sizes(case, seed=cut)
    tame(b)
    e = torch.full(tuple(b.vs.shape), float(last))
    for t in b.tables:
        e[t[:cut]] = float(first)
    b.vs = powers(e)
    b.check(status)


def leaning(case, lean, seed=0):
    """Keys of the first half of each context score ``lean`` (in powers of two) more than those of the second, which all rows see alike."""
    b = sizes(case, seed=seed)
    k = torch.zeros(tuple(b.k.shape))
    for t, ctx in zip(b.tables, b.ctx_lens):
        half = t[:-(-ctx // b.page // 2)]
        k[half, :, :, 0] = 1
        k[half, :, :, 1] = torch.randn((len(half), b.page, b.kv), generator=torch.Generator().manual_seed(seed)) * 0.01
    b.k = k.to(E4M3).cuda()
    b.ks.fill_(1)
    b.q.fill_(0)
    b.q[:, :, 0], b.q[:, :, 1] = 4.0, 1.0
    b.scale = lean * math.log(2) / 4
    return b


@pytest.mark.parametrize("case", SPLIT, ids=name_of)
@pytest.mark.parametrize("lean,near,far", [(30, -40, 0), (60, -40, 0), (60, -110, -20), (-30, 0, -40), (-30, 0, -20), (150, -100, 100), (-150, 100, -100), (200, -100, 100), (20, -12, 12), (40, 0, 0)])
def test_weights_against_scales(status, case, lean, near, far):  # noqa: F811
    """The half that has the weight has the small scales: the product of the two decides, whichever it favours."""
    b = leaning(case, lean)
    e = torch.full(tuple(b.vs.shape), float(far))
    for t, ctx in zip(b.tables, b.ctx_lens):
        e[t[:-(-ctx // b.page // 2)]] = float(near)
    b.vs = powers(e)
    b.check(status)


@pytest.mark.parametrize("case", SPLIT, ids=name_of)
@pytest.mark.parametrize("small", [-20, -100])
def test_pages_of_zeros_between_small_ones(status, case, small):  # noqa: F811
    """Values of zero have the scale 0, which says nothing of the others'."""
    b = sizes(case, seed=2)
    e = torch.full(tuple(b.vs.shape), float(small))
    b.vs = powers(e)
    for t in b.tables:
        b.vs[t[1::3]] = 0
        b.vs[t[-1]] = 0
    b.check(status)
    b.vs.zero_()
    got = b.run(status)
    fine(status)
    assert bool((got == 0).all())


@pytest.mark.parametrize("case", SPLIT, ids=name_of)
def test_later_pages_do_not_touch_the_rows_before_them(status, case):  # noqa: F811
    """Some tokens of a portion lie on a page that the tokens before them do not see; its scales may be anything."""
    b = sizes(case, page=8, seed=5)
    at = b.q_lens[0]                                 # request 1
    seen = b.ctx_lens[1] // 8 * 8 if b.ctx_lens[1] % 8 else b.ctx_lens[1] - 8
    rows = seen - (b.ctx_lens[1] - b.q_lens[1])      # of its tokens before the last page
    e = torch.full(tuple(b.vs.shape), -30.0)
    for last in (-30, 60, -90):
        e[b.tables[1][-1]] = float(last)
        b.vs = powers(e)
        got = b.run(status)
        fine(status)
        want, spread, size = P.attention(b.q, b.k.float(), b.v.float(), b.ks, b.vs, b.q_lens, b.ctx_lens, b.tables, b.scale)
        tol = P.tolerance(want, spread, size, b.dtype, b.d, max(b.ctx_lens))
        off = (got.double().cpu() - want).abs()
        assert bool((off[at:at + rows] <= tol[at:at + rows]).all()) and bool((off <= tol).all())


@pytest.mark.parametrize("case", SPLIT, ids=name_of)
def test_scales_of_any_sign_and_mantissa(status, case):  # noqa: F811
    b = sizes(case, seed=6)
    gen = torch.Generator().manual_seed(6)
    b.ks *= 0.5 + torch.rand(b.ks.shape, generator=gen).cuda()
    b.vs *= (0.5 + torch.rand(b.vs.shape, generator=gen)).cuda() * torch.where(torch.rand(b.vs.shape, generator=gen) < 0.3, -1.0, 1.0).cuda()
    b.ks[b.tables[0][2]] *= -1
    b.check(status)
    b.vs[b.tables[0][1]] = 1e-41        # below float32's normal range
    b.vs[b.tables[0][3]] = 1.7 * 2.0 ** 126
    got = b.run(status).double().cpu()
    fine(status)
    want, spread, size = P.attention(b.q, b.k.float(), b.v.float(), b.ks, b.vs, b.q_lens, b.ctx_lens, b.tables, b.scale)
    tol = P.tolerance(want, spread, size, b.dtype, b.d, max(b.ctx_lens))
    # codes of up to 448 times that scale: some results are rounded to infinity, and one within half a step of the border to either side of it
    most = torch.finfo(b.dtype).max
    beyond, inside = want.abs() > most * (1 + torch.finfo(b.dtype).eps / 2) + tol, want.abs() < most - tol
    assert bool(beyond.any()) and bool(((got - want).abs() <= tol)[inside].all())
    assert torch.equal(got[beyond], torch.copysign(torch.tensor(math.inf, dtype=torch.float64), want[beyond]))


@pytest.mark.parametrize("case", SPLIT, ids=name_of)
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_a_scale_that_is_no_number_reaches_the_rows_that_see_it(status, case, odd):  # noqa: F811
    """However little weight its keys have; the rows before its page do not notice."""
    b = leaning(case, 140)
    page = b.tables[1][-1]              # the last keys of request 1, of next to no weight
    first = (len(b.tables[1]) - 1) * b.page
    want = b.run(status)
    b.vs[page, 1] = odd
    got = b.run(status)
    fine(status)
    at = b.q_lens[0]
    for i in range(sum(b.q_lens)):
        pos = b.ctx_lens[1] - b.q_lens[1] + i - at
        if i < at or pos < first:
            assert torch.equal(got[i], want[i])
        else:
            assert torch.equal(got[i, :2], want[i, :2]) and not bool(torch.isfinite(got[i, 2:]).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [144, 192, 224])
def test_head_sizes_above_128(status, dtype, d):  # noqa: F811
    """Rows of keys that are an odd number of 16-byte words, and panels of 64 and 32 bytes; ordinary scales, and ones far apart."""
    b = Batch([1, 3, 0, 9], [90, 33, 5, 170], heads=6, kv=2, d=d, page=16, dtype=dtype, seed=d)
    b.check(status)
    b.check(status, window=20)
    tame(b)
    b.vs = powers(torch.randint(LOWEST, HIGHEST + 1, b.vs.shape, generator=torch.Generator().manual_seed(d)))
    b.check(status)


@pytest.mark.parametrize("page", [1, 8, 24, 48])
@pytest.mark.parametrize("far", [False, True])
def test_pages_of_other_sizes(status, page, far):  # noqa: F811
    """A scale for each key, pages that end inside a block of keys; scales that one walk is enough for and ones that make a warp begin anew."""
    b = Batch([1, 4], [700, 330], heads=8, kv=2, d=64, page=page, dtype=torch.bfloat16, seed=page)
    gen = torch.Generator().manual_seed(page)
    b.vs = powers(torch.randint(-70, 20, b.vs.shape, generator=gen) if far else torch.randint(-3, 2, b.vs.shape, generator=gen))
    b.check(status)
    b.check(status, window=100)


def test_one_page_among_many_makes_its_warp_begin_anew(status):  # noqa: F811
    """The others' stretches are joined to its: sums with a power of two beside them and sums without."""
    for dtype in DTYPES:
        for at in (0, 40, 90, 124):
            b = Batch([1, 1], [2000, 1500], heads=8, kv=2, d=128, page=16, dtype=dtype, seed=at)
            tame(b)
            b.vs.fill_(2.0 ** -8)
            b.vs[b.tables[0][at]] = 2.0 ** 100
            b.vs[b.tables[1][min(at, 93)]] = 2.0 ** -110
            b.check(status)
            want = b.run(status)
            assert all(torch.equal(b.run(status), want) for _ in range(5))


@pytest.mark.parametrize("case", SPLIT, ids=name_of)
@pytest.mark.parametrize("lean", [0, 30, 50, 70, -20])
@pytest.mark.parametrize("zeros", ["first", "last", "all"])
def test_blocks_of_zeros(status, case, lean, zeros):  # noqa: F811
    """Half of a context, or all of it, holds nothing but zeros, with scales of 0: its keys have their weights all the same."""
    b = leaning(case, lean)
    e = torch.full(tuple(b.vs.shape), -6.0)
    b.vs = powers(e)
    for t, ctx in zip(b.tables, b.ctx_lens):
        cut = -(-ctx // b.page // 2)
        b.vs[t if zeros == "all" else t[:cut] if zeros == "first" else t[cut:]] = 0
    b.check(status)
    if zeros == "all":
        assert bool((b.run(status) == 0).all())
