"""The 8-bit cache where other tests do not look: the engine's codes from bfloat16, chained launches, long portions of float32 queries."""

import pytest
import torch

import util
from plain import kv8_plain as P
from test_kv8_engine import folders, runner  # noqa: F401
from test_kv8_gpu import Batch, status  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["A", "B"])
def test_the_first_layers_cache_holds_the_rounded_bfloat16_keys_and_values(folders, name):  # noqa: F811
    """Layer 0's keys and values do not depend on the cache: codes and scales are bit by bit those of the bfloat16 cache's contents, stored in the same portions."""
    from oxr_inference_b200.engine.batch import StepEntry

    ids, cuts = util.token_ids(name, 50, seed=6), [13, 1, 1, 30, 5]
    held = {}
    for kv in ("auto", "e4m3"):
        r = runner(folders[name], name, "bfloat16", kv)
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
    assert table == table8 and plain.k_pools[0].dtype == torch.bfloat16
    slots = [table[p // page] * page + p % page for p in range(len(ids))]
    for pool, codes, scales in ((plain.k_pools[0], eight.k_pools[0], eight.scales[0][0]), (plain.v_pools[0], eight.v_pools[0], eight.scales[0][1])):
        x = pool[0].flatten(0, 1)[slots].cpu()
        want = (torch.zeros(codes[0].shape), torch.zeros(scales[0].shape))
        at = 0
        for c in cuts:
            want = P.store(x[at:at + c], slots[at:at + c], *want)
            at += c
        assert torch.equal(codes[0].float().double().cpu(), want[0]) and torch.equal(scales[0].double().cpu(), want[1])


CONFIG = {"architectures": ["Qwen3ForCausalLM"], "model_type": "qwen3", "hidden_size": 4096, "intermediate_size": 12288, "num_hidden_layers": 2,
          "num_attention_heads": 32, "num_key_value_heads": 8, "head_dim": 128, "rms_norm_eps": 1e-6, "rope_theta": 1000000.0, "vocab_size": 2048,
          "tie_word_embeddings": False, "max_position_embeddings": 8192}


@pytest.mark.parametrize("requests", [1, 13])
def test_replays_of_a_decode_step_agree_however_its_kernels_overlap(requests):
    """A step over an 8-bit cache, on the same state: kernels that start while the one before still runs give the bits of kernels launched one behind the other."""
    from oxr_inference_b200 import ops
    from oxr_inference_b200.engine.batch import StepEntry
    from oxr_inference_b200.engine.graphs import DecodeGraphs
    from oxr_inference_b200.engine.runtime import ModelRunner
    from oxr_inference_b200.ops import kv8

    class Graphs(DecodeGraphs):
        def _forward(self, ctx):
            self.logits = self.runner.model.step(ctx, self.runner.cache)
            s = ctx.sampling
            return ops.sample(self.logits, s["temperature"], s["seed_lo"], s["seed_hi"], s["counter"])

    made = ModelRunner.from_config(CONFIG, 1, dtype="bfloat16", page_size=16, num_pages=1200, max_requests=requests, max_positions=8192, kv_cache_dtype="e4m3")
    entries = []
    for i in range(requests):
        request = made.cache.open(i)
        length = 200 + 1600 * i // max(requests - 1, 1)
        assert made.cache.reserve(request, length + 1)
        made.step([StepEntry(request, [(7 * i + 31 * p) % 2048 for p in range(length)], [])])
        entries.append(StepEntry(request, [i], [0]))
    cold = torch.empty(64 << 20, device="cuda")
    libs = [ops._lib(), kv8._kv8_lib(128)]
    want = None
    try:
        for chained in (1, 0):
            for lib in libs:
                lib.oxr_set_chain(chained)
            graphs = Graphs(made, max_batch=requests, max_positions=8192)
            for _ in range(40 if chained else 2):
                cold.fill_(1.0)
                torch.cuda.synchronize()
                graphs.run(entries)
                torch.cuda.synchronize()
                got = graphs.logits[:requests].clone()
                want = got if want is None else want
                assert torch.equal(got, want)
    finally:
        for lib in libs:
            lib.oxr_set_chain(int(ops.CHAIN_KERNELS))
    made.check()


@pytest.mark.parametrize("heads,kv,d,page", [(8, 2, 128, 16), (4, 4, 64, 24), (6, 2, 256, 16)])
@pytest.mark.parametrize("window", [0, 60])
def test_long_portions_of_float32_queries(status, heads, kv, d, page, window):  # noqa: F811
    Batch([200, 1, 90], [333, 400, 90], heads=heads, kv=kv, d=d, page=page, dtype=torch.float32, seed=d).check(status, window=window)


@pytest.mark.parametrize("d,group", [(144, 2), (256, 4)])
def test_long_portions_of_heads_above_128(status, d, group):  # noqa: F811
    Batch([150, 33], [300, 33], heads=2 * group, kv=2, d=d, page=16, dtype=torch.bfloat16, seed=d).check(status)
