"""Decoding several tokens with no host work between the steps, against steps that the host builds one by one."""

import pytest
import torch

import util

pytestmark = pytest.mark.gpu


def make(folder, name, dtype, kv="auto", pages=60, page=None):
    from oxr_inference_b200.engine.runtime import ModelRunner

    return ModelRunner.from_folder(folder, dtype=dtype, page_size=page or util.PAGE.get(name, 8), num_pages=pages, max_requests=5, kv_cache_dtype=kv)


def begin(r, prompts):
    """The prompts in the cache, and the first token of each."""
    from oxr_inference_b200.engine.batch import StepEntry

    caches = [r.cache.open() for _ in prompts]
    for rc, p in zip(caches, prompts):
        assert r.cache.reserve(rc, len(p))
    logits = r.step([StepEntry(rc, p, [len(p) - 1]) for rc, p in zip(caches, prompts)])
    return caches, logits.argmax(-1).tolist()


def one_by_one(r, caches, tokens, steps):
    from oxr_inference_b200.engine.batch import StepEntry

    out = [[] for _ in caches]
    for _ in range(steps):
        for rc in caches:
            assert r.cache.reserve(rc, rc.length + 1)
        tokens = r.step([StepEntry(rc, [t], [0]) for rc, t in zip(caches, tokens)]).argmax(-1).tolist()
        for o, t in zip(out, tokens):
            o.append(t)
    r.check()
    return out


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("device_decode")
    return {name: util.make_folder(tmp, name, seed=7) for name in ("A", "B")}


@pytest.mark.parametrize("name,kv", [("A", "auto"), ("B", "auto"), ("A", "e4m3"), ("B", "e4m3")])
def test_the_tokens_of_steps_built_by_the_host(folders, name, kv):
    """Across pages, behind a window that gives pages back (B), more steps than are kept on the GPU at a time; and the requests go on either way."""
    prompts = [util.token_ids(name, n, seed=30 + n) for n in (3, 16, 41)]
    r = make(folders[name], name, "float32", kv)
    caches, tokens = begin(r, prompts)
    want = one_by_one(r, caches, tokens, 90)
    s = make(folders[name], name, "float32", kv)
    caches2, tokens2 = begin(s, prompts)
    assert tokens2 == tokens
    got = s.decode(caches2, tokens2, 5)
    got = [g + h for g, h in zip(got, s.decode(caches2, [g[-1] for g in got], 70))]
    got = [g + h for g, h in zip(got, one_by_one(s, caches2, [g[-1] for g in got], 15))]
    assert got == want
    assert [rc.length for rc in caches2] == [rc.length for rc in caches]
    s.cache.check()


def test_bfloat16_and_other_requests_between(folders):
    """The graph is used again for other requests with other pages; those that are not decoded keep what they have."""
    r = make(folders["A"], "A", "bfloat16")
    prompts = [util.token_ids("A", n, seed=50 + n) for n in (20, 5, 33)]
    caches, tokens = begin(r, prompts)
    first = r.decode(caches[:2], tokens[:2], 9)
    last = r.decode(caches[1:], [first[1][-1], tokens[2]], 20)
    assert len(r._device_decode._loops) == 1
    other = make(folders["A"], "A", "bfloat16")
    alone, same = begin(other, prompts[2:])
    assert same == tokens[2:]
    # bfloat16 products depend on the number of rows in their last bits: a near tie may fall the other way, after which the sequences differ
    want = other.decode(alone, same, 20)[0]
    assert last[1][:3] == want[:3] and all(len(x) == 20 for x in last)


def test_a_model_with_state_beside_its_pages(tmp_path):
    import radapel_util

    folder = radapel_util.make_folder(tmp_path, radapel_util.MODEL_X, "x", 3)
    r, s = (make(folder, "radapel", "float32", page=8) for _ in range(2))
    prompts = [[5, 17, 3, 9, 11, 2, 8, 1, 4], [9, 8, 7]]
    caches, tokens = begin(r, prompts)
    caches2, tokens2 = begin(s, prompts)
    assert s.decode(caches2, tokens2, 21) == one_by_one(r, caches, tokens, 21)


def test_refusals(folders):
    r = make(folders["A"], "A", "float32", pages=8)
    caches, tokens = begin(r, [util.token_ids("A", 20, seed=1), util.token_ids("A", 9, seed=2)])
    free = r.cache.free_pages
    for requests, given, steps in (([], [], 3), (caches, tokens[:1], 3), (caches, tokens, 0), (caches[:1] * 2, tokens, 3), (caches, tokens, 600)):
        with pytest.raises(ValueError):
            r.decode(requests, given, steps)
    with pytest.raises(RuntimeError, match="lacks pages"):
        r.decode(caches, tokens, 100)
    assert r.cache.free_pages == free and [rc.length for rc in caches] == [20, 9]
    assert len(r.decode(caches, tokens, 4)[0]) == 4
