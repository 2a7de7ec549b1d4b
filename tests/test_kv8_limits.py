"""Sizes of 8-bit pools that the entry points refuse because numbers of 32 bits do not count them; without a GPU."""

import pytest
import torch

from oxr_inference_b200 import ops
from test_kv8_rules import E4M3, INT, on_cpu  # noqa: F401


def far_pools(pages, page, kv, d):
    k = torch.empty((pages, page, kv, d), dtype=E4M3, device="meta")
    s = torch.empty((pages, kv), device="meta")
    return k, k, s, s


@pytest.mark.parametrize("pages,page,kv,d", [(1 << 31, 1, 1, 16), (1, 1 << 31, 1, 16), (1, 1, 1 << 27, 16)])
def test_pools_beyond_32_bits_are_refused(on_cpu, pages, page, kv, d):  # noqa: F811
    pools = far_pools(pages, page, kv, d)
    meta = dict(device="meta")
    x = torch.empty((1, kv, d), **meta)
    one, status = torch.empty(1, dtype=INT, **meta), torch.empty(4, dtype=INT, **meta)
    with pytest.raises(ops.KernelError, match="32 bits"):
        ops.store_kv8(x, x, one, *pools, status)
    with pytest.raises(ops.KernelError, match="32 bits"):
        ops.paged_attention_kv8(x, *pools, cu_q=torch.empty(2, dtype=INT, **meta), ctx_lens=one, block_table=torch.empty((1, 1), dtype=INT, **meta), scale=1.0, max_q_len=1,
                                kv_len_bound=1, status=status)


def test_long_pages_are_refused_with_the_settings(monkeypatch):
    """Not by the store, in the first step."""
    import finolix_util
    from oxr_inference_b200.config import EngineSettings
    from oxr_inference_b200.engine import runtime

    assert EngineSettings(page_size=8192, kv_cache_dtype="e4m3").page_size == ops.KV8_LONGEST_PAGE
    assert EngineSettings(page_size=8193).page_size == 8193
    with pytest.raises(ValueError, match="page_size 8193"):
        EngineSettings(page_size=8193, kv_cache_dtype="e4m3")
    monkeypatch.setattr(runtime, "require_cuda", lambda device: torch.device("cpu"))
    monkeypatch.setattr(runtime.ops, "new_status", lambda device: torch.zeros(4, dtype=INT))
    with pytest.raises(ValueError, match="page_size 8193"):
        runtime.ModelRunner.build_model(finolix_util.MODEL_A, None, dtype="bfloat16", page_size=8193, kv_cache_dtype="e4m3")
