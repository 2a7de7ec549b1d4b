"""Attention of long portions over the 8-bit cache (the tcgen05 kernel) against plain 64-bit arithmetic."""

import math

import pytest
import torch

from oxr_inference_b200.ops import kv8
from plain import kv8_plain as P
from test_kv8_gpu import Batch, fine, ints, status  # noqa: F401

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def small_steps_too(monkeypatch):
    """The kernel is for steps of many tiles; what it computes does not depend on how many there are."""
    monkeypatch.setattr(kv8, "kv8_prompt_pays", lambda *a: True)


def batch(q_lens, ctx_lens, **kw):
    kw = {"heads": 32, "kv": 8, "d": 128, "page": 16, "dtype": BF16, **kw}
    b = Batch(q_lens, ctx_lens, **kw)
    assert kv8.kv8_prompt_takes(max(q_lens), b.d, BF16, b.scale), "the case does not reach the kernel"
    return b


@pytest.mark.parametrize("heads,kv,d,page", [(32, 8, 128, 16), (12, 12, 64, 32), (24, 12, 80, 24), (12, 12, 16, 8), (36, 12, 48, 7), (60, 12, 112, 1), (13, 13, 96, 300), (12, 12, 32, 16)])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_sizes(status, heads, kv, d, page, window):  # noqa: F811
    """Portions that begin inside a block of keys and end inside a tile; beside them requests that the other kernel takes."""
    batch([70, 1, 9, 0, 33, 8], [301, 77, 9, 0, 128, 60], heads=heads, kv=kv, d=d, page=page).check(status, window=window)


@pytest.mark.parametrize("q_len,ctx", [(65, 65), (65, 200), (128, 128), (129, 1000), (257, 257), (300, 1111)])
def test_one_request_of_several_tiles(status, q_len, ctx):  # noqa: F811
    batch([q_len], [ctx]).check(status)


@pytest.mark.parametrize("heads,kv,d", [(300, 12, 16), (600, 2, 16), (48, 3, 64)])
def test_large_groups_of_heads(status, heads, kv, d):  # noqa: F811
    """25, 16 and 300 query heads on a KV head: rows of one token in both halves, a second tile for one KV head's heads."""
    batch([60, 20], [90, 20], heads=heads, kv=kv, d=d, peak=1.0).check(status)


def test_rows_that_see_nothing_are_zero(status):  # noqa: F811
    b = batch([100, 70, 40], [60, 0, 40])
    b.check(status)
    got = b.run(status)
    assert bool((got[:40] == 0).all()) and bool((got[100:170] == 0).all()) and bool((got[40] != 0).any())


@pytest.mark.parametrize("window", [0, 20])
def test_what_is_hidden_may_hold_anything(status, window):  # noqa: F811
    b = batch([70, 90], [150, 90], d=64, seed=2)
    for r, ctx in enumerate(b.ctx_lens):
        for o in range(ctx % 16, 16):
            b.k.view(torch.uint8)[b.tables[r][-1], o] = 0x7F
            b.v.view(torch.uint8)[b.tables[r][-1], o] = 0xFF
    spare = [p for p in range(b.k.shape[0]) if all(p not in t for t in b.tables)]
    b.ks[spare], b.vs[spare] = math.nan, math.inf
    if window:   # pages before every window of request 0
        b.k.view(torch.uint8)[b.tables[0][0]] = 0x7F
        b.v.view(torch.uint8)[b.tables[0][1]] = 0x7F
        b.ks[b.tables[0][0]], b.vs[b.tables[0][1]] = math.nan, math.inf
    b.check(status, window=window)
    # NaN in one entry of a late token's value: earlier tokens must not notice, later ones that see it get it
    at, pos = 70 + 60, 60
    want = b.run(status, window=window)
    b.v.view(torch.uint8)[b.tables[1][pos // 16], pos % 16, 2, 5] = 0x7F
    got = b.run(status, window=window)
    fine(status)
    assert torch.equal(got[:at], want[:at])
    end = 160 if not window else min(160, at + window)
    assert bool(torch.isnan(got[at:end, 8:12, 5]).all())
    assert torch.equal(got[end:], want[end:])
    clean = torch.ones(64, dtype=torch.bool)
    clean[5] = False
    assert torch.equal(got[at:][:, :, clean], want[at:][:, :, clean]) and torch.equal(got[at:, :8], want[at:, :8])
    # a whole value scale: the rows that see a token of its page
    b.v.view(torch.uint8)[b.tables[1][pos // 16], pos % 16, 2, 5] = 0
    b.vs[b.tables[1][4], 3] = math.nan   # positions 64 to 79
    got = b.run(status, window=window)
    fine(status)
    assert torch.equal(got[:70 + 60], want[:70 + 60]) and bool(torch.isnan(got[70 + 64:70 + 80, 12:16]).all())


@pytest.mark.parametrize("exponents", [(-118, -118), (100, 100), (-60, 20), (0, 0)])
def test_scales_of_any_size(status, exponents):  # noqa: F811
    b = batch([70, 40], [200, 75], seed=3)
    gen = torch.Generator().manual_seed(1)
    e = torch.randint(exponents[0], exponents[1] + 1, b.vs.shape, generator=gen).float()
    b.vs = torch.ldexp(torch.ones_like(e), e.int()).cuda()
    b.ks *= 1.37       # all scales by one factor: their ratios are powers of two all the same
    if exponents == (0, 0):
        b.vs[b.tables[0][0]] = 0
        b.vs[b.tables[1]] = 0
        b.ks[b.tables[0][3]] = 0
    b.check(status)


def test_scales_that_are_no_powers_of_two(status):  # noqa: F811
    """The ratio of two scales, and a code times it, are then rounded to fp16: half a step is 2^-11 of a number, twice in every key and value."""
    b = batch([70, 40], [200, 75], seed=4)
    gen = torch.Generator().manual_seed(2)
    b.ks *= 0.5 + torch.rand(b.ks.shape, generator=gen).cuda()
    b.vs *= 0.5 + torch.rand(b.vs.shape, generator=gen).cuda()
    got = b.run(status)
    fine(status)
    want, spread, size = P.attention(b.q, b.k.float(), b.v.float(), b.ks, b.vs, b.q_lens, b.ctx_lens, b.tables, b.scale)
    # a score moves by 2 x 2^-11 of its magnitudes at most, which moves numerator and denominator; a value by as much of itself
    tol = P.tolerance(want, spread, size, BF16, b.d, 200) + (4 * 2.0 ** -11 * size + 2 * 2.0 ** -11) * spread
    assert bool(((got.double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("factor", [1e-30, 1e-3, 40.0])
def test_queries_of_any_size(status, factor):  # noqa: F811
    b = batch([70, 40], [300, 65], seed=5)
    b.q = (b.q.float() * factor).to(BF16)
    b.check(status)


def test_nan_queries_reach_their_rows_alone(status):  # noqa: F811
    b = batch([70, 40], [90, 40])
    want = b.run(status)
    b.q[17, 1, 3] = math.nan
    got = b.run(status)
    fine(status)
    assert bool(torch.isnan(got[17, 1]).all())
    got[17, 1] = want[17, 1]
    assert torch.equal(got, want)


def test_strides_out_and_rows_behind(status):  # noqa: F811
    b = batch([70, 4, 20], [160, 35, 90], heads=16, kv=16, d=64, seed=6)
    want = b.run(status)
    both = torch.stack([b.k.view(torch.uint8), b.v.view(torch.uint8)], 1).view(b.k.dtype)
    b.k, b.v = both[:, 0], both[:, 1]
    wide = torch.full((99, 18 * 64), math.nan, dtype=BF16, device="cuda")
    wide[:94, 64:64 * 17] = b.q.flatten(1)
    out = torch.full((99, 16, 64), 7.0, dtype=BF16, device="cuda")
    got = b.run(status, q=wide[:, 64:64 * 17].unflatten(1, (16, 64)), out=out)
    fine(status)
    assert got is out and torch.equal(got[:94], want) and bool((got[94:] == 7).all())


def test_bad_pages_and_lengths_are_reported(status):  # noqa: F811
    b = batch([70, 70], [90, 90])
    want = b.run(status)
    table = b.table.clone()
    for bad in (-1, b.k.shape[0], 1 << 30):
        b.table[1, 1] = bad
        got = b.run(status)
        torch.cuda.synchronize()
        assert status.tolist()[0] == 4 and torch.equal(got[:70], want[:70])
        status.zero_()
    b.table = table
    b.ctx = ints([90, 97])
    b.run(status)
    torch.cuda.synchronize()
    assert status.tolist()[0] == 4
    status.zero_()
    b.ctx = ints([90, 90])
    b.run(status, max_q_len=69)
    torch.cuda.synchronize()
    assert status.tolist()[0] == 100
    status.zero_()


def test_replayed_and_on_two_streams(status):  # noqa: F811
    b = batch([70, 1, 100], [700, 90, 133])
    want = b.run(status)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(10):
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


def test_a_request_alone_with_fewer_tokens_than_its_bound(status):  # noqa: F811
    """What a graph captured for the largest portion sees when it is replayed for a small one."""
    b = batch([100], [300])
    b.check(status)
    for q in (1, 5, 64):
        small = Batch([q], [300 - 7 * q], heads=32, kv=8, d=128, page=16, dtype=BF16, seed=q)
        small.check(status, max_q_len=100)
