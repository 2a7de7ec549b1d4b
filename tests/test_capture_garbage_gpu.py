"""Captures of decode steps while there is garbage that holds CUDA graphs, and what keeps graphs alive."""

import gc
import weakref

import pytest
import torch

import util
from test_device_decode_gpu import begin, folders, make  # noqa: F401

pytestmark = pytest.mark.gpu


class Circle:
    """Goes when garbage is collected, and a captured graph with it."""

    def __init__(self):
        self.me = self
        x = torch.ones(1 << 20, device="cuda")
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.out = x + 1


def used_runner(folder):
    """One that has decoded, in a circle too: graphs that were replayed, pinned memory that copies have read, pools."""
    r = make(folder, "A", "float32")
    caches, tokens = begin(r, [util.token_ids("A", 9, seed=3), util.token_ids("A", 4, seed=4)])
    r.decode(caches, tokens, 3)
    r.decode(caches[:1], tokens[:1], 3)
    r.me = r
    return r


def with_garbage(model, stock):
    """Every step of the model lets go of a circle first, in the capture too, and the collector runs if it may."""
    step = model.step

    def stepped(*args):
        if stock:
            stock.pop()
        if gc.isenabled():
            gc.collect()
        return step(*args)

    model.step = stepped


def test_a_capture_on_the_way_to_decoding_on_the_gpu(folders):  # noqa: F811
    prompts = [util.token_ids("A", n, seed=90 + n) for n in (9, 14)]
    r, s = (make(folders["A"], "A", "float32") for _ in range(2))
    (caches, tokens), (caches2, tokens2) = begin(r, prompts), begin(s, prompts)
    want = r.decode(caches, tokens, 5)
    stock = [made() for made in (Circle, lambda: used_runner(folders["A"])) for _ in range(2)]
    with_garbage(s.model, stock)
    assert s.decode(caches2, tokens2, 5) == want
    assert len(stock) == 2 and gc.isenabled()     # an eager step first, then the capture


def test_captures_of_an_engine(folders):  # noqa: F811
    from oxr_inference_b200 import Engine, EngineSettings, SamplingParams

    prompts = [util.token_ids("A", n, seed=95 + n) for n in (5, 12, 7)]

    def engine():
        return Engine(folders["A"], EngineSettings(dtype="float32", page_size=util.PAGE["A"], num_pages=40, max_running=3))

    params = SamplingParams(max_tokens=6, ignore_eos=True)
    want = [c.token_ids for c in engine().generate(prompts, params)]
    made = engine()
    stock = [used_runner(folders["A"]) if i % 3 else Circle() for i in range(12)]
    with_garbage(made.runner.model, stock)
    assert [c.token_ids for c in made.generate(prompts, params)] == want
    assert made.counters["graph_steps"] > 0 and gc.isenabled()


def test_a_runner_goes_with_its_last_name(folders):  # noqa: F811
    """Its graphs, weights and pools do not wait for the collector."""
    r = make(folders["A"], "A", "float32")
    caches, tokens = begin(r, [util.token_ids("A", 9, seed=3)])
    assert len(r.decode(caches, tokens, 3)[0]) == 3
    gone = weakref.ref(r)
    gc.collect()
    gc.disable()
    try:
        del r
        assert gone() is None
    finally:
        gc.enable()
