"""8-bit pools whose pages, scales or rows lie beyond what 32 bits count: the results are those of the same entries in small pools."""

import pytest
import torch

from test_kv8_gpu import E4M3, Batch, fine, ints, status  # noqa: F401

pytestmark = pytest.mark.gpu
INT = torch.int32


def room(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB of device memory")


@pytest.fixture
def many_scales():
    """More than 2^31 scales: pages of one token with two heads of 16. Keys and values share their memory, and hold the same."""
    room(64)
    pages, kv, d = (1 << 30) + 64, 2, 16
    codes = torch.empty((pages, 1, kv, d), dtype=torch.uint8, device="cuda").view(E4M3)
    scales = torch.empty((pages, kv), device="cuda")
    yield codes, scales
    del codes, scales
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_where_the_scales_are_more_than_2_to_the_31(status, many_scales, dtype):  # noqa: F811
    codes, scales = many_scales
    b = Batch([1, 2], [50, 37], heads=4, kv=2, d=16, page=1, dtype=dtype, seed=1)
    b.v, b.vs = b.k, b.ks
    want = b.run(status)
    small = b.k.shape[0]
    at = codes.shape[0] - small       # the last pages; their scales' places are above 2^31
    codes.view(torch.uint8)[at:] = b.k.view(torch.uint8)
    scales[at:] = b.ks
    b.k = b.v = codes
    b.ks = b.vs = scales
    b.table = torch.where(b.table >= 0, b.table + at, b.table).to(INT)
    got = b.run(status)
    fine(status)
    assert torch.equal(got, want)


@pytest.mark.parametrize("n", [40, 1300])
def test_store_where_the_pages_are_more_than_2_to_the_30(status, many_scales, n):  # noqa: F811
    """Both forms of the store: few tokens, and many, for which it keeps two words a page."""
    from oxr_inference_b200 import ops

    codes, scales = many_scales
    gen = torch.Generator().manual_seed(2)
    x = torch.randn((n, 2, 16), generator=gen).to("cuda", torch.bfloat16)
    small = 1400
    slots = torch.randperm(small, generator=gen)[:n].to("cuda", INT)
    k = torch.zeros((small, 1, 2, 16), dtype=torch.uint8, device="cuda").view(E4M3)
    ks = torch.zeros((small, 2), device="cuda")
    ops.store_kv8(x, x, slots, k, k.clone(), ks, ks.clone(), status)
    at = codes.shape[0] - small
    codes.view(torch.uint8)[at:] = 0
    scales[at:] = 0
    ops.store_kv8(x, x, (slots + at).to(INT), codes, codes, scales, scales, status)
    fine(status)
    assert torch.equal(codes.view(torch.uint8)[at:], k.view(torch.uint8)) and torch.equal(scales[at:], ks)


@pytest.mark.parametrize("pays", [False, True])
def test_pages_of_more_than_2_to_the_31_bytes(status, pays, monkeypatch):  # noqa: F811
    """The last tokens of such a page, seen through a window; both kernels."""
    from oxr_inference_b200.ops import kv8

    monkeypatch.setattr(kv8, "kv8_prompt_pays", lambda *a: pays)
    room(12)
    page, kv, d, q_len, window = (1 << 24) + 9, 8, 16, 12, 40
    b = Batch([q_len], [256 - 3], heads=16, kv=kv, d=d, page=257, dtype=torch.bfloat16, seed=3, spare=0)
    want = b.run(status, window=window)
    far = (1 << 24) - 3                # the same place in a block of keys
    code = torch.empty((2, page, kv, d), dtype=torch.uint8, device="cuda")
    for i, c in enumerate((b.k, b.v)):
        code[i, far - 200:far] = c.view(torch.uint8)[0, 253 - 200:253]
    b.k, b.v = code[:1].view(E4M3), code[1:].view(E4M3)
    b.ctx = ints([far])
    got = b.run(status, window=window, kv_len_bound=far)
    fine(status)
    assert torch.equal(got, want)
    del code
    b.k = b.v = None
    torch.cuda.empty_cache()
