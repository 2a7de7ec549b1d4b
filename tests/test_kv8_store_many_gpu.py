"""The store of more than 1,024 tokens, which finds its pages by a kernel of its own, by the rules of the one for few."""

import math
import random

import pytest
import torch

from plain import kv8_plain as P
from test_kv8_gpu import E4M3, check_store, fine, ints, normal, same_codes, status  # noqa: F401

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
SIZES = [(16, 2, 16), (24, 3, 80), (16, 2, 128), (64, 1, 128), (7, 1, 256), (100, 2, 48)]   # pages whose entries are held in registers and ones that are not


def shuffled(pages, page, n, seed):
    """Slots of ``n`` tokens in any order: pages in several runs, some slots twice, some tokens skipped."""
    rng = random.Random(seed)
    slots = rng.sample(range(pages * page), n)
    for _ in range(40):
        slots[rng.randrange(n)] = slots[rng.randrange(n)]
    for _ in range(30):
        slots[rng.randrange(n)] = rng.choice([-1, -2, -(1 << 31)])
    return slots


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,kv,d", SIZES)
def test_any_order_slots_twice_and_growing_scales(status, dtype, page, kv, d):  # noqa: F811
    pages = 2400 // page
    n = 1300
    a, b = shuffled(pages, page, n, page), shuffled(pages, page, n, page + 1)
    check_store(status, n_pages=pages, page=page, kv=kv, d=d, dtype=dtype, calls=[(normal(1), a), (normal(2, 9.0), b), (normal(3, 1e-3), a[::-1])], gap=16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,kv,d", SIZES)
def test_portions_of_prompts(status, dtype, page, kv, d):  # noqa: F811
    """Requests of some pages each that begin and end inside a page; then the next portion of each."""
    rng = random.Random(d)
    pages = 3400 // page
    order = rng.sample(range(pages), pages)
    first, second, at = [], [], 0
    while at < pages and len(first) < 1500:
        own = order[at:at + 7]
        at += 7
        slots = [p * page + o for p in own for o in range(page)]
        cut = rng.randrange(len(slots) // 2, len(slots))
        first += slots[:cut]
        second += slots[cut:]
    assert len(first) > 1024
    check_store(status, n_pages=pages, page=page, kv=kv, d=d, dtype=dtype, calls=[(normal(4), first), (normal(5, 3.0), second)])


def test_extremes_among_many(status):  # noqa: F811
    """Infinities, NaN, zeros and the ends of the range; powers of two at the border."""
    n, page = 1200, 4
    gen = torch.Generator().manual_seed(6)

    def odd(m, w):
        x = torch.randn((m, w), generator=gen) * torch.exp2(torch.randint(-120, 120, (m, 1), generator=gen).float())
        x[::7] = 0
        x[3::31, 0], x[5::31, 1], x[7::31, 2] = math.inf, -math.inf, math.nan
        x[9::31] = 448 * torch.exp2(torch.randint(-90, 90, (x[9::31].shape[0], 1), generator=gen).float())
        x[11::31] = -1e-44
        return x

    slots = random.Random(7).sample(range(400 * page), n)
    check_store(status, n_pages=400, page=page, kv=2, d=16, dtype=torch.float32, calls=[(odd, slots), (odd, slots[::-1])])


@pytest.mark.parametrize("n", [1025, 2000])
def test_slots_outside_are_reported_and_the_rest_is_stored(status, n):  # noqa: F811
    from oxr_inference_b200 import ops

    pages, page, kv, d = 150, 16, 2, 32
    slots = shuffled(pages, page, n, n)
    for i, bad in ((0, pages * page), (n // 2, pages * page + 5), (n - 1, (1 << 31) - 1)):
        slots[i] = bad
    x = normal(8)(n, kv * d).view(n, kv, d).to("cuda", torch.bfloat16)
    pools = [torch.zeros((pages, page, kv, d), device="cuda").to(E4M3) for _ in range(2)]
    scales = [torch.zeros((pages, kv), device="cuda") for _ in range(2)]
    ops.store_kv8(x, x, ints(slots), *pools, *scales, status)
    torch.cuda.synchronize()
    assert status.tolist()[0] == 2 and status.tolist()[1] in (0, n // 2, n - 1)
    codes, want = P.store(x.cpu(), slots, torch.zeros((pages, page, kv, d)), torch.zeros((pages, kv)))
    for i in range(2):
        assert torch.equal(scales[i].double().cpu(), want)
        same_codes(pools[i], codes)


def test_two_streams_have_scratch_of_their_own(status):  # noqa: F811
    """Stores of many tokens into two caches at a time, and replayed from a graph."""
    from oxr_inference_b200 import ops

    pages, page, kv, d, n = 200, 16, 2, 64, 2500
    made = []
    for i in range(2):
        x = normal(10 + i)(n, kv * d).view(n, kv, d).to("cuda", torch.bfloat16)
        made.append((x, ints(shuffled(pages, page, n, i)), torch.zeros((pages, page, kv, d), device="cuda").to(E4M3), torch.zeros((pages, kv), device="cuda")))

    def into(i, pool, scale):
        x, slots, _, _ = made[i]
        ops.store_kv8(x, x, slots, pool, pool.clone(), scale, scale.clone(), status)

    want = []
    for i in range(2):
        pool, scale = made[i][2].clone(), made[i][3].clone()
        into(i, pool, scale)
        want.append((pool, scale))
    fine(status)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for r in range(12):
        with torch.cuda.stream(streams[r % 2]):
            pool, scale = made[r % 2][2].clone(), made[r % 2][3].clone()
            into(r % 2, pool, scale)
            got.append((pool, scale))
    fine(status)
    for r, (pool, scale) in enumerate(got):
        assert torch.equal(pool.view(torch.uint8), want[r % 2][0].view(torch.uint8)) and torch.equal(scale, want[r % 2][1])
    pool, scale = made[0][2].clone(), made[0][3].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        into(0, pool, scale)
    pool.view(torch.uint8).zero_()
    scale.zero_()
    graph.replay()
    fine(status)
    assert torch.equal(pool.view(torch.uint8), want[0][0].view(torch.uint8)) and torch.equal(scale, want[0][1])
