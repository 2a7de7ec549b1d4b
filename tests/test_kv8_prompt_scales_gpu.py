"""Attention of long portions over 8-bit pages whose scales are far apart (the tcgen05 kernel), by the tests of the split-key one."""

import math

import pytest
import torch

import test_kv8_scales_gpu as S
from oxr_inference_b200.ops import kv8
from plain import kv8_plain as P
from test_kv8_gpu import Batch, fine, status  # noqa: F401

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
CASES = [("d64", BF16, 64, [70, 20], [330, 150]), ("d128", BF16, 128, [100, 30], [270, 400])]
by_size = pytest.mark.parametrize("case", CASES, ids=[c[0] for c in CASES])


@pytest.fixture(autouse=True)
def small_steps_too(monkeypatch):
    monkeypatch.setattr(kv8, "kv8_prompt_pays", lambda *a: True)


@by_size
@pytest.mark.parametrize("seed", range(16))
def test_value_scales_over_all_that_the_store_makes(status, case, seed):  # noqa: F811
    S.test_value_scales_over_all_that_the_store_makes(status, case, seed)


@by_size
@pytest.mark.parametrize("first,last", [(S.LOWEST, 12), (12, S.LOWEST), (5, S.LOWEST), (S.LOWEST, S.HIGHEST), (S.HIGHEST, S.LOWEST), (-40, 40), (40, -40), (0, 5), (5, 0), (0, 3), (3, 0)])
@pytest.mark.parametrize("cut", [1, 4, 9, 12])
def test_two_value_scales(status, case, first, last, cut):  # noqa: F811
    S.test_two_value_scales(status, case, first, last, min(cut, 9))


@by_size
@pytest.mark.parametrize("lean,near,far", [(30, -40, 0), (60, -40, 0), (60, -110, -20), (-30, 0, -40), (-30, 0, -20), (150, -100, 100), (-150, 100, -100), (200, -100, 100), (20, -12, 12), (40, 0, 0),
                                           (90, -59, 50), (-90, 50, -59)])
def test_weights_against_scales(status, case, lean, near, far):  # noqa: F811
    S.test_weights_against_scales(status, case, lean, near, far)


@by_size
@pytest.mark.parametrize("small", [-20, -100])
def test_pages_of_zeros_between_small_ones(status, case, small):  # noqa: F811
    S.test_pages_of_zeros_between_small_ones(status, case, small)


@by_size
def test_later_pages_do_not_touch_the_rows_before_them(status, case):  # noqa: F811
    S.test_later_pages_do_not_touch_the_rows_before_them(status, case)


@by_size
def test_scales_of_any_sign_and_mantissa(status, case):  # noqa: F811
    S.test_scales_of_any_sign_and_mantissa(status, case)


@by_size
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_a_scale_that_is_no_number_reaches_the_rows_that_see_it(status, case, odd):  # noqa: F811
    S.test_a_scale_that_is_no_number_reaches_the_rows_that_see_it(status, case, odd)


@by_size
@pytest.mark.parametrize("seed", range(10))
@pytest.mark.parametrize("low,high", [(-60, 20), (-24, 0), (-16, 0), (-4, 0)])
def test_key_and_value_scales_apart(status, case, seed, low, high):  # noqa: F811
    """Keys too: a page whose keys are next to nothing still has its place among the scores."""
    b = S.sizes(case, seed=seed, peak=1.0)
    gen = torch.Generator().manual_seed(seed)
    b.vs = S.powers(torch.randint(low, high + 1, b.vs.shape, generator=gen))
    b.ks = S.powers(torch.randint(max(low, -30), high + 1, b.ks.shape, generator=gen).clamp(max=-6))
    b.check(status)


@by_size
def test_a_small_page_with_all_the_weight_beside_a_large_one(status, case):  # noqa: F811
    """In one block of keys: the page that the queries look at has values 2^-40 of the size of its neighbours', whose keys have 2^-80 of its weight."""
    b = S.sizes(case, seed=8)
    k = torch.full(tuple(b.k.shape), 0.0)
    k[..., 0] = -1
    for t in b.tables:
        k[t[2], :, :, 0] = 1
    b.k = k.to(b.k.dtype).cuda()
    b.ks.fill_(1)
    b.q.fill_(0)
    b.q[:, :, 0] = 4
    b.scale = 10 * math.log(2)
    e = torch.zeros(tuple(b.vs.shape))
    for t in b.tables:
        e[t[2]] = -40
    b.vs = S.powers(e)
    b.check(status)
    got = b.run(status).float()
    fine(status)
    assert bool((got != 0).any()) and float(got.abs().max()) < 2.0 ** -30


@pytest.mark.parametrize("seed", range(4))
def test_rows_differ_in_what_they_see(status, seed):  # noqa: F811
    """A prompt from its first token on, pages of eight: each row sees other scales; with and without a window."""
    b = Batch([150], [150], heads=8, kv=2, d=64, page=8, dtype=BF16, seed=seed)
    S.tame(b)
    gen = torch.Generator().manual_seed(seed)
    low, high = ((S.LOWEST, S.HIGHEST), (-40, 40), (-10, 10), (-3, 3))[seed]
    b.vs = S.powers(torch.randint(low, high + 1, b.vs.shape, generator=gen))
    b.ks = S.powers(torch.randint(-12, -6, b.ks.shape, generator=gen))
    b.check(status)
    b.check(status, window=30)
    # what comes later changes nothing but the last bits of what is before it
    at = 96
    want, spread, size = P.attention(b.q, b.k.float(), b.v.float(), b.ks, b.vs, b.q_lens, b.ctx_lens, b.tables, b.scale)
    tol = P.tolerance(want, spread, size, BF16, b.d, 150)[:at]
    for later in (-118, 0, 120):
        b.vs[b.tables[0][at // 8:]] = 2.0 ** later
        got = b.run(status).double().cpu()[:at]
        fine(status)
        assert bool(((got - want[:at]).abs() <= tol).all())


def test_a_build_that_cannot_run_the_kernel_leaves_its_steps_to_the_other(status, monkeypatch):  # noqa: F811
    b = S.sizes(CASES[1], seed=1)
    monkeypatch.setattr(kv8, "kv8_prompt_runs", lambda d: False)
    b.check(status)
    got = b.run(status)
    monkeypatch.setattr(kv8, "kv8_prompt_pays", lambda *a: False)
    assert torch.equal(b.run(status), got)
    monkeypatch.undo()
    assert kv8.kv8_prompt_runs(128) and kv8.kv8_prompt_runs(16) and not kv8.kv8_prompt_runs(144)


@by_size
@pytest.mark.parametrize("lean", [0, 30, 50, 70, -20])
@pytest.mark.parametrize("zeros", ["first", "last", "all"])
def test_blocks_of_zeros(status, case, lean, zeros):  # noqa: F811
    S.test_blocks_of_zeros(status, case, lean, zeros)


def any_mantissa(b, seed):
    gen = torch.Generator().manual_seed(seed)
    b.ks *= 1 + torch.rand(b.ks.shape, generator=gen).cuda()
    b.vs = (0.01 * (1 + 3 * torch.rand(b.vs.shape, generator=gen))).cuda()


@by_size
@pytest.mark.parametrize("seed", range(6))
def test_scales_of_any_mantissa_within_2_to_the_4(status, case, seed):  # noqa: F811
    """As a cache has them whose scales are a page's largest magnitude over 448. (A rounded ratio or product, 2^-11 of a score, would show.)"""
    b = S.sizes(case, seed=seed, peak=6.0)
    any_mantissa(b, seed)
    b.check(status)
    b.check(status, window=70)
    b.ks[b.tables[0][3]] *= -1
    b.ks[b.tables[1][2]] = 0
    b.check(status)


@by_size
def test_values_of_zero_beside_key_scales_of_any_mantissa(status, case):  # noqa: F811
    b = S.sizes(case, seed=3)
    any_mantissa(b, 3)
    b.vs.zero_()
    got = b.run(status)
    fine(status)
    assert bool((got == 0).all())


@by_size
@pytest.mark.parametrize("power", [60, 70, 100, -100])
def test_large_key_scales_and_small_queries(status, case, power):  # noqa: F811
    b = S.sizes(case, seed=4)
    any_mantissa(b, 4)
    b.q = (b.q.float() * 2.0 ** -power).to(BF16)
    b.ks *= 2.0 ** power
    b.check(status)
    b.ks = S.powers(torch.full(tuple(b.ks.shape), power - 8.0))       # the same with keys that are powers of two
    b.check(status)


@by_size
def test_mixed_kinds_of_blocks(status, case):  # noqa: F811
    """Powers of two, any mantissas and scales far apart, 128 keys each and across."""
    b = S.sizes(case, seed=5)
    gen = torch.Generator().manual_seed(5)
    for t in b.tables:
        for i, p in enumerate(t):
            kind = (i // 5) % 3
            b.vs[p] = 0.01 * float(1 + torch.rand((), generator=gen)) if kind == 1 else 2.0 ** int(torch.randint(*((-7, -5) if kind == 0 else (-70, 20)), (), generator=gen))
            b.ks[p] *= 1.0 if kind == 0 else float(1 + torch.rand((), generator=gen))
    b.check(status)
    b.check(status, window=90)
