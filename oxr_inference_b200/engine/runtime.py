"""Builds the model, its cache and its step function from a model folder or a configuration."""

from __future__ import annotations

import gc
from contextlib import contextmanager
from pathlib import Path
from typing import Any, Iterator, Mapping

import torch

from oxr_inference_b200 import ops
from oxr_inference_b200.cache.manager import CacheManager, RequestCache
from oxr_inference_b200.config.model_config import read_config_json
from oxr_inference_b200.config.registry import resolve_architecture
from oxr_inference_b200.engine.batch import BatchBuilder, StepEntry
from oxr_inference_b200.parts.base import Runtime
from oxr_inference_b200.parts.decoder import DecoderModel
from oxr_inference_b200.weights.loader import load_weights, tensor_shapes
from oxr_inference_b200.weights.random_init import fill_random

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32, "bf16": torch.bfloat16, "fp32": torch.float32}


def require_cuda(device: str | torch.device = "cuda") -> torch.device:
    device = torch.device(device)
    if device.type != "cuda" or not torch.cuda.is_available():
        raise RuntimeError("this engine runs on a CUDA device only (sm_100a kernels, no CPU path); "
                           f"asked for {device}, torch.cuda.is_available() = {torch.cuda.is_available()}")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    # Matrix products of the 32-bit path and the fp32 accumulation of the 16-bit path are to be exact.
    torch.backends.cuda.matmul.allow_tf32 = False
    torch.backends.cuda.matmul.allow_bf16_reduced_precision_reduction = False
    return device


@contextmanager
def no_collection() -> Iterator[None]:
    """Garbage stays where it is while a CUDA graph is captured: what it frees on the GPU (another graph, in the first place) would make the capture invalid."""
    was = gc.isenabled()
    gc.disable()
    try:
        yield
    finally:
        if was:
            gc.enable()


class ModelRunner:
    """A model with its weights, its cache and its step function: what generation and trace replay both drive."""

    def __init__(self, model: DecoderModel, config: Any, *, page_size: int, num_pages: int, max_requests: int):
        self.model, self.config = model, config
        rt = model.runtime
        if rt.page_size != page_size:
            raise ValueError(f"the model was built for pages of {rt.page_size} tokens, the cache is asked for {page_size}")
        ops.warm_up(model.head_dims())
        self.cache = CacheManager(model.cache_plan, page_size=page_size, num_pages=num_pages, max_requests=max_requests,
                                  device=rt.device, dtype=rt.dtype)
        self.builder = BatchBuilder(self.cache, model.tile_specs, rt.device, rt.status)
        self.steps = 0
        self._device_decode = None

    # ---- construction
    @staticmethod
    def build_model(raw_config: Mapping[str, Any], generation: Mapping[str, Any] | None, *, dtype: str,
                    device: str | torch.device = "cuda", max_positions: int | None = None, page_size: int = 16,
                    kv_cache_dtype: str = "auto", shapes: Mapping[str, tuple[int, ...]] | None = None):
        """``shapes``: the checkpoint's tensor shapes, for designs that leave a size to them (``Architecture.shapes_matter``)."""
        dev = require_cuda(device)
        arch = resolve_architecture(raw_config)
        config = arch.config_from_dict(raw_config, generation)
        spec = arch.spec_for(config, shapes)
        runtime = Runtime(device=dev, dtype=DTYPES[dtype], max_positions=max_positions or spec.max_positions,
                          status=ops.new_status(dev), page_size=page_size, kv_dtype=kv_cache_dtype)
        if kv_cache_dtype == "e4m3" and page_size > ops.KV8_LONGEST_PAGE:
            raise ValueError(f"page_size {page_size}: pages of 8-bit keys and values hold up to {ops.KV8_LONGEST_PAGE} tokens")
        model = DecoderModel(spec, runtime)
        if kv_cache_dtype != "auto" and not any(g.need.eight_bit for g in model.cache_plan.groups):
            raise ValueError(f"kv_cache_dtype {kv_cache_dtype!r}: no layer of this model keeps keys and values that could be held in 8 bits")
        return model, config

    @classmethod
    def from_folder(cls, model_dir: str | Path, *, dtype: str, page_size: int, num_pages: int, max_requests: int,
                    device: str | torch.device = "cuda", max_positions: int | None = None, kv_cache_dtype: str = "auto") -> "ModelRunner":
        raw, generation = read_config_json(model_dir)
        arch = resolve_architecture(raw)
        model, config = cls.build_model(raw, generation, dtype=dtype, device=device, max_positions=max_positions, page_size=page_size,
                                        kv_cache_dtype=kv_cache_dtype, shapes=tensor_shapes(model_dir) if arch.shapes_matter else None)
        load_weights(model, model_dir)
        return cls(model, config, page_size=page_size, num_pages=num_pages, max_requests=max_requests)

    @classmethod
    def from_config(cls, raw_config: Mapping[str, Any], seed: int, *, dtype: str, page_size: int, num_pages: int,
                    max_requests: int, device: str | torch.device = "cuda", max_positions: int | None = None,
                    std: float = 0.02, norm_std: float = 0.1, kv_cache_dtype: str = "auto") -> "ModelRunner":
        """Random weights drawn on the device (no file)."""
        model, config = cls.build_model(raw_config, None, dtype=dtype, device=device, max_positions=max_positions, page_size=page_size,
                                        kv_cache_dtype=kv_cache_dtype)
        fill_random(model, seed, std=std, norm_std=norm_std)
        return cls(model, config, page_size=page_size, num_pages=num_pages, max_requests=max_requests)

    # ---- the step function
    @torch.inference_mode()
    def step(self, entries: list[StepEntry], *, advance: bool = True) -> torch.Tensor:
        """Run one batch of (request, its next tokens): prompt portions beside single decoded tokens, cut anywhere.

        Only the given tokens are computed, against the cache earlier steps left; their keys and values are added
        to it. Pages for them must have been reserved (``cache.reserve``). Returns fp32 logits
        ``[sum(len(e.want)), vocab]`` in entry order, then ``want`` order. With ``advance`` each request's cached
        length moves forward and pages a window has passed are released."""
        if not entries:
            raise ValueError("a step needs at least one entry")
        ctx = self.builder.build(entries)
        logits = self.model.step(ctx, self.cache)
        if advance:
            for e in entries:
                self.cache.advance(e.cache, e.cache.length + len(e.tokens))
        self.steps += 1
        return logits

    def decode(self, requests: list[RequestCache], tokens: list[int], steps: int) -> list[list[int]]:
        """The next ``steps`` tokens of each request, chosen greedily on the GPU with no host work between the steps (see :class:`DeviceDecode`);
        ``tokens``: the last token of each, not yet in its cache."""
        from oxr_inference_b200.engine.device_decode import DeviceDecode

        if self._device_decode is None:
            self._device_decode = DeviceDecode(self)
        return self._device_decode.run(requests, tokens, steps)

    def check(self) -> None:
        """Raise if any kernel reported an error since the last check (synchronises)."""
        ops.check_status(self.model.runtime.status)
