"""What the entry points of the 8-bit cache refuse and how they cut the work, without a GPU."""

import pytest
import torch

from oxr_inference_b200 import ops
from oxr_inference_b200.ops import kv8
from plain import kv8_plain as P

E4M3 = torch.float8_e4m3fn
INT = torch.int32


@pytest.fixture
def on_cpu(monkeypatch):
    """Lets CPU tensors through to the checks behind that of the device; whatever passes them all would reach a library."""
    def never(*a, **k):
        raise AssertionError("a call that should have been refused reached the library")

    monkeypatch.setattr(kv8, "_here", lambda t, name: None)
    monkeypatch.setattr(kv8, "_kv8_lib", never)
    monkeypatch.setattr(kv8, "_core_lib", never)


def pools(pages=3, page=16, kv=2, d=32):
    k, v = (torch.zeros((pages, page, kv, d)).to(E4M3) for _ in range(2))
    return k, v, torch.zeros((pages, kv)), torch.zeros((pages, kv))


def status():
    return torch.zeros(4, dtype=INT)


def test_cpu_tensors_are_refused():
    x = torch.zeros((1, 2, 32))
    with pytest.raises(ops.KernelError, match="CUDA device only"):
        ops.store_kv8(x, x, torch.zeros(1, dtype=INT), *pools(), status())
    with pytest.raises(ops.KernelError, match="CUDA device only"):
        ops.paged_attention_kv8(x, *pools(), cu_q=torch.zeros(2, dtype=INT), ctx_lens=torch.zeros(1, dtype=INT), block_table=torch.zeros((1, 1), dtype=INT), scale=1.0,
                                max_q_len=1, kv_len_bound=1, status=status())
    one = torch.zeros(1, dtype=INT)
    with pytest.raises(ops.KernelError, match="CUDA device only"):
        ops.step_pages(one, one, torch.zeros((1, 1), dtype=INT), one, one, one, page_size=16, tokens=1, status=status())


def bad_pools():
    k, v, ks, vs = pools()
    wide = torch.zeros((3, 16, 2, 64)).to(E4M3)
    odd = torch.zeros(3 * 16 * 2 * 32 + 8).to(E4M3)[8:].view(3, 16, 2, 32)
    return {
        "another type": (k.float(), v, ks, vs), "other sizes": (k, pools(pages=4)[1], ks, vs), "parts of rows": (wide[..., :32], wide[..., :32], ks, vs),
        "pages apart differently": (torch.zeros((3, 2, 16, 2, 32)).to(E4M3)[:, 0], v, ks, vs), "head size": (*pools(d=24)[:2], ks, vs),
        "not aligned": (odd if odd.data_ptr() % 16 else odd.flatten()[8:], v, ks, vs), "scales of another type": (k, v, ks.double(), vs),
        "scales of other sizes": (k, v, ks, vs[:2]), "scales with strides": (k, v, ks, torch.zeros((3, 4))[:, ::2]), "three dimensions": (k[0], v[0], ks, vs),
        "no pages": pools(pages=0), "no places": pools(page=0),
    }


@pytest.mark.parametrize("name", sorted(bad_pools()))
def test_bad_pools(on_cpu, name):
    p = bad_pools()[name]
    x = torch.zeros((1, 2, 32))
    with pytest.raises(ops.KernelError):
        ops.store_kv8(x, x, torch.zeros(1, dtype=INT), *p, status())
    with pytest.raises(ops.KernelError):
        ops.paged_attention_kv8(x, *p, cu_q=torch.zeros(2, dtype=INT), ctx_lens=torch.zeros(1, dtype=INT), block_table=torch.zeros((1, 1), dtype=INT), scale=1.0,
                                max_q_len=1, kv_len_bound=1, status=status())


def test_bad_stores(on_cpu):
    x, slots = torch.zeros((4, 2, 32)), torch.zeros(4, dtype=INT)
    for k, v, s in ((x[:3], x, slots), (x, x[:, :1], slots), (x, x.bfloat16(), slots), (x.half(), x.half(), slots), (x, x, slots.long()), (x, x, slots[::2]),
                    (x[..., ::2], x[..., ::2], slots), (x, x, slots.view(2, 2)), (torch.zeros((4, 2, 36))[..., :32], x, slots),
                    (torch.zeros((4, 66))[:, 1:65].unflatten(1, (2, 32)), x, slots)):
        with pytest.raises(ops.KernelError):
            ops.store_kv8(k, v, s, *pools(), status())
    with pytest.raises(ops.KernelError):
        ops.store_kv8(x, x, slots, *pools(page=8200, pages=1), status())
    with pytest.raises(ops.KernelError):
        ops.store_kv8(x, x, slots, *pools(), status().long())


def test_bad_attention_calls(on_cpu):
    good = dict(q=torch.zeros((3, 4, 32)), cu_q=torch.zeros(3, dtype=INT), ctx_lens=torch.zeros(2, dtype=INT), block_table=torch.zeros((2, 5), dtype=INT), scale=1.0,
                window=0, max_q_len=2, kv_len_bound=10, status=status(), out=None)

    def call(**change):
        how = {**good, **change}
        return ops.paged_attention_kv8(how.pop("q"), *pools(), **how)

    for change in (dict(q=torch.zeros((3, 3, 32))), dict(q=torch.zeros((3, 4, 16))), dict(q=torch.zeros((3, 4, 32)).half()), dict(q=torch.zeros((3, 0, 32))),
                   dict(q=torch.zeros((3, 128))), dict(q=torch.zeros((3, 4, 64))[..., ::2]), dict(cu_q=torch.zeros(2, dtype=INT)), dict(cu_q=torch.zeros(3)),
                   dict(ctx_lens=torch.zeros(3, dtype=INT)), dict(block_table=torch.zeros((3, 5), dtype=INT)), dict(block_table=torch.zeros(5, dtype=INT)),
                   dict(block_table=torch.zeros((2, 10), dtype=INT)[:, ::2]), dict(window=-1), dict(max_q_len=0), dict(out=torch.zeros((2, 4, 32))),
                   dict(out=torch.zeros((3, 4, 32)).bfloat16()), dict(out=torch.zeros((3, 4, 64))[..., :32])):
        with pytest.raises(ops.KernelError):
            call(**change)
    both = torch.zeros((5, 4, 32))
    for q, out in ((both[:3], both[:3]), (both[1:4], both[2:5]), (torch.zeros((3, 6, 32))[:, :4], None)):
        if out is None:      # columns of a wider product; its memory as output
            out = torch.as_strided(q, (3, 4, 32), (128, 32, 1))
        with pytest.raises(ops.KernelError, match="over q"):
            call(q=q, out=out)
    # nothing to do: no library is needed
    assert call(q=torch.zeros((0, 4, 32))).shape == (0, 4, 32)
    out = torch.full((3, 4, 32), 5.0)
    assert call(cu_q=torch.zeros(1, dtype=INT), ctx_lens=torch.zeros(0, dtype=INT), block_table=torch.zeros((0, 5), dtype=INT), out=out) is out and bool((out == 5).all())


def test_bad_tables(on_cpu):
    row = torch.zeros(3, dtype=INT)
    good = dict(lengths=row, held=row, block_table=torch.zeros((3, 4), dtype=INT), free_list=torch.zeros(9, dtype=INT), free_count=torch.zeros(1, dtype=INT), q_lens=row,
                fresh=None, page_size=16, tokens=5, status=status())
    for change in (dict(lengths=row[:2]), dict(held=row.long()), dict(q_lens=torch.zeros(4, dtype=INT)), dict(fresh=row[:1]), dict(fresh=row.bool()), dict(page_size=0),
                   dict(tokens=-1), dict(free_count=row), dict(free_list=torch.zeros((3, 3), dtype=INT)), dict(block_table=row),
                   dict(block_table=torch.zeros((3, 8), dtype=INT)[:, ::2]), dict(page_size=1 << 29), dict(page_size=1 << 28), dict(tokens=1 << 30)):
        with pytest.raises(ops.KernelError):
            ops.step_pages(**{**good, **change})
    many = torch.zeros(8193, dtype=INT)
    with pytest.raises(ops.KernelError):
        ops.step_pages(many, many, torch.zeros((8193, 1), dtype=INT), good["free_list"], good["free_count"], many, page_size=16, tokens=1, status=status())


def test_who_can_do_a_step():
    bf16 = torch.bfloat16
    assert kv8.kv8_prompt_takes(2048, 128, bf16, 0.1) and kv8.kv8_prompt_takes(9, 16, bf16, 1e-9)
    for most, d, dtype, scale in ((2048, 128, torch.float32, 0.1), (2048, 256, bf16, 0.1), (2048, 128, bf16, 0.0), (2048, 128, bf16, -0.1), (8, 128, bf16, 0.1)):
        assert not kv8.kv8_prompt_takes(most, d, dtype, scale)


@pytest.mark.parametrize("requests,q,seen,heads,kv,d,pays", [(1, 2048, 4096, 32, 8, 128, True), (1, 64, 4096, 32, 8, 128, False), (1, 128, 8192, 32, 8, 128, False),
                                                            (1, 256, 4096, 32, 8, 128, True), (16, 16, 2048, 32, 8, 128, True), (1, 512, 512, 32, 8, 128, True),
                                                            (1, 256, 4096, 8, 8, 128, False), (1, 2048, 8192, 8, 1, 128, True), (16, 25, 552, 16, 2, 64, False)])
def test_who_is_faster(requests, q, seen, heads, kv, d, pays):
    """The sides that were measured to be."""
    assert kv8.kv8_prompt_pays(requests, requests * q, q, heads, kv, d, seen) == pays


def test_blocks():
    assert kv8.kv8_blocks(8, 64, 444) == 128 and kv8.kv8_blocks(512, 64, 444) == 444 and kv8.kv8_blocks(1, 1, 444) == 1


def test_plain_codes_are_torchs():
    gen = torch.Generator().manual_seed(1)
    x = torch.cat([torch.randn(4000, generator=gen) * 10 ** torch.randint(-4, 3, (4000,), generator=gen), torch.tensor([448.0, -448.0, 0.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -10])])
    x = x.clamp(-448, 448)
    assert torch.equal(P.e4m3(x), x.to(E4M3).double())
    assert [P.scale_for(s) for s in (0.0, 448.0, 448.0001, 7.0, 1e-40)] == [0.0, 1.0, 2.0, 2.0 ** -6, 2.0 ** -118]


def test_plain_pages_give_back_and_take():
    held, table, stack, count, begin, cu = P.pages([20, 5], [2, 1], [[7, 8, -1], [9, -1, -1]], ([3, 4, -1, -1, -1], 2), [1, 30], [1, 0], 16)
    assert (held, begin, cu, count) == ([1, 3], [0, 5], [0, 1, 31], 1)
    assert table[0][0] == 8 and table[1] == [9, 7, 4] and stack[:1] == [3]


def test_pools_of_more_slots_than_there_are_numbers(on_cpu):
    pages = (1 << 27) - 511      # of 16 tokens: 2^31 - 8176 slots
    k, v, scales = torch.empty((pages, 16, 1, 16), dtype=E4M3, device="meta"), torch.empty((pages, 16, 1, 16), dtype=E4M3, device="meta"), torch.empty((pages, 1), device="meta")
    x, slots = (torch.empty((1, 1, 16), device="meta"), torch.empty(1, dtype=INT, device="meta"))
    with pytest.raises(ops.KernelError, match="slots below"):
        ops.store_kv8(x, x, slots, k, v, scales, scales, torch.empty(4, dtype=INT, device="meta"))
    # one page less: with no tokens there is nothing left to do
    ops.store_kv8(x[:0], x[:0], slots[:0], k[1:], v[1:], scales[1:], scales[1:], torch.empty(4, dtype=INT, device="meta"))
