"""The engine with keys and values cached in 8 bits."""

import pytest
import torch

import util
from oxr_inference_b200.cache import CacheManager, make_cache_plan
from oxr_inference_b200.config import EngineSettings
from oxr_inference_b200.parts.base import PagedKVNeed
from plain import kv8_plain as P
from plain import qwen3_plain as QP


def test_settings():
    assert EngineSettings().kv_cache_dtype == "auto" and EngineSettings(kv_cache_dtype="e4m3").kv_cache_dtype == "e4m3"
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        EngineSettings(kv_cache_dtype="fp4")


def test_bytes_of_a_page():
    """A byte an entry and two scales per KV head; groups of other needs beside it as before."""
    plan = make_cache_plan([PagedKVNeed(8, 128, eight_bit=True)] * 3 + [PagedKVNeed(8, 128)], [None] * 4)
    assert len(plan.groups) == 2
    assert CacheManager.bytes_per_page(plan, 16, torch.bfloat16) == 3 * 8 * (2 * 16 * 128 + 8) + 2 * 8 * 16 * 128 * 2


def test_pools_and_views():
    plan = make_cache_plan([PagedKVNeed(2, 32, eight_bit=True)] * 3 + [PagedKVNeed(2, 32, 8)], [None] * 4)
    m = CacheManager(plan, page_size=4, num_pages=5, max_requests=2, device=torch.device("cpu"), dtype=torch.bfloat16)
    view = m.group_view(0, torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    assert view.k_pool.dtype == torch.float8_e4m3fn and view.k_pool.shape == (3, 5, 4, 2, 32) and view.k_scale.shape == view.v_scale.shape == (3, 5, 2)
    other = m.group_view(1, torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    assert other.k_pool.dtype == torch.bfloat16 and other.k_scale is None
    assert m.group_view(0, view.block_table, view.slots).k_scale is m.scales[0][0]


# ------------------------------------------------------------------------------------------------------------------ on the GPU
@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("kv8")
    return {name: util.make_folder(tmp, name, seed=5) for name in ("A", "B")}


def eight_bit_logits(folder, ids, page, monkeypatch):
    """The plain implementation's logits with every layer's keys and values rounded as the cache holds them when all tokens come in one step."""
    plain = QP.causal_attention

    def through_the_cache(q, k, v, scale, window=0):
        n, kv, d = k.shape
        pages = -(-n // page)
        rounded = []
        for x in (k, v):
            codes, scales = P.store(x, list(range(n)), torch.zeros((pages, page, kv, d)), torch.zeros((pages, kv)))
            rounded.append((codes * scales[:, None, :, None]).flatten(0, 1)[:n].to(x.dtype))
        return plain(q, *rounded, scale, window)

    cfg, w = QP.read_model(folder, torch.float32)
    with monkeypatch.context() as m:
        m.setattr(QP, "causal_attention", through_the_cache)
        return QP.logits(cfg, w, ids)


def runner(folder, name, dtype, kv="e4m3", pages=64):
    from oxr_inference_b200.engine.runtime import ModelRunner

    return ModelRunner.from_folder(folder, dtype=dtype, page_size=util.PAGE[name], num_pages=pages, max_requests=3, kv_cache_dtype=kv)


def run_portions(r, ids, cuts):
    from oxr_inference_b200.engine.batch import StepEntry

    rc = r.cache.open()
    out, at = [], 0
    for c in cuts:
        assert r.cache.reserve(rc, at + c)
        out.append(r.step([StepEntry(rc, ids[at:at + c], list(range(c)))]))
        at += c
    r.check()
    r.cache.close(rc)
    return torch.cat(out).float().cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_are_those_of_a_rounded_cache(folders, name, dtype, monkeypatch):
    """Whole prompts, portions and single tokens, with a windowed layer whose pages go to other requests (B).

    A code can come out one step away where the engine's fp32 key differs from the plain one in its last bits; with some 10^4 codes and 10^-6 between the two that
    is one code or none, whose effect is a few hundredths of what rounding all of them by a third of a step does. Portions differ from a whole prompt in
    the scales of the moment only, which power-of-two scales let no code above e4m3's subnormal range notice. So a fifth of the difference that 8 bits make
    bounds float32. A bfloat16 key is off by up to 2^-8 and what its layer's input is off by (1 to 2 in a hundred), a good part of a code's step of 2^-4 to
    2^-3 of it, so many codes come out apart: between the two lie the rounding of one side, the rounding of the other and bfloat16's own 3 in a hundred
    (util.compare)."""
    n = 131
    ids = util.token_ids(name, n, seed=4)
    want = eight_bit_logits(folders[name], ids, util.PAGE[name], monkeypatch)
    effect = (want - util.plain_logits(folders[name], ids)).pow(2).mean().sqrt()
    r = runner(folders[name], name, dtype)
    for cuts in ([n], [40, 17, 3, 71], [n - 20] + [1] * 20):
        got = run_portions(r, ids, cuts)
        if dtype == "float32":
            assert (got - want).pow(2).mean().sqrt() <= 0.2 * effect, cuts
        else:
            assert (got - want).pow(2).mean().sqrt() <= 2 * effect + 3e-2 * want.pow(2).mean().sqrt(), cuts
    r.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "B"])
def test_the_first_layers_cache_holds_the_rounded_keys_and_values(folders, name):
    """Layer 0's keys and values do not depend on the cache: its codes and scales are those of the 32-bit cache's contents, stored in the same portions."""
    from oxr_inference_b200.engine.batch import StepEntry

    ids, cuts = util.token_ids(name, 50, seed=6), [13, 1, 1, 30, 5]
    held = {}
    for kv in ("auto", "e4m3"):
        r = runner(folders[name], name, "float32", kv)
        rc = r.cache.open()
        at = 0
        for c in cuts:
            assert r.cache.reserve(rc, at + c)
            r.step([StepEntry(rc, ids[at:at + c], [c - 1])])
            at += c
        r.check()
        held[kv] = (r.cache, rc.tables[0][:])
    page = util.PAGE[name]
    (plain, table), (eight, table8) = held["auto"], held["e4m3"]
    assert table == table8
    slots = [table[p // page] * page + p % page for p in range(len(ids))]
    for pool, codes, scales in ((plain.k_pools[0], eight.k_pools[0], eight.scales[0][0]), (plain.v_pools[0], eight.v_pools[0], eight.scales[0][1])):
        x = pool[0].flatten(0, 1)[slots].cpu()
        want = (torch.zeros(codes[0].shape), torch.zeros(scales[0].shape))
        at = 0
        for c in cuts:
            want = P.store(x[at:at + c], slots[at:at + c], *want)
            at += c
        assert torch.equal(codes[0].float().double().cpu(), want[0]) and torch.equal(scales[0].double().cpu(), want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "B"])
def test_graphs_and_page_pressure_change_no_token(folders, name):
    """Requests that come and go with few pages (pages pass from one to another, some requests are begun again), decoded from graphs and without them."""
    from oxr_inference_b200 import Engine, SamplingParams

    prompts = [util.token_ids(name, n, seed=20 + n) for n in (3, 30, 17, 45, 8, 26)]
    got = {}
    for graphs in (True, False):
        engine = Engine(folders[name], EngineSettings(dtype="float32", kv_cache_dtype="e4m3", page_size=util.PAGE[name], num_pages=16 if name == "A" else 24, max_running=3,
                                                      cuda_graphs=graphs, prefill_chunk=19, max_step_tokens=32))
        got[graphs] = [c.token_ids for c in engine.generate(prompts, SamplingParams(max_tokens=12, ignore_eos=True))]
        if graphs:
            assert engine.counters["graph_steps"] > 0
    assert got[True] == got[False] and all(len(t) == 12 for t in got[True])


@pytest.mark.gpu
def test_a_model_without_such_layers_is_refused():
    import finolix_util
    from oxr_inference_b200.engine.runtime import ModelRunner

    with pytest.raises(ValueError, match="kv_cache_dtype"):
        ModelRunner.build_model(finolix_util.MODEL_A, None, dtype="bfloat16", kv_cache_dtype="e4m3")


@pytest.mark.gpu
def test_command_line(folders, capsys):
    from oxr_inference_b200.__main__ import main

    assert main(["--model", str(folders["A"]), "--prompt-ids", "5,17,3", "--max-tokens", "4", "--num-pages", "16", "--kv-cache-dtype", "e4m3", "--ignore-eos"]) == 0
    assert '"token_ids"' in capsys.readouterr().out
