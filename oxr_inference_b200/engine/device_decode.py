"""Several decode steps of the same requests without the host between them.

The reference's decode loop comes back to the host after every token: it copies the chosen tokens out, works out slots and lengths, and
copies them in again (oxr_runtime/decode_graph.py:102-115, oxr_runtime/engine.py:557-608). Here one CUDA graph holds a whole step that
feeds itself: ``ops.step_pages`` works out positions, slots and boundaries from the lengths of the requests, the layers run, the token of
the largest logit is chosen and becomes the next step's input, the lengths move on. The host reserves the pages for all steps, replays the
graph once per step and reads the tokens at the end.
"""

from __future__ import annotations

import weakref
from dataclasses import dataclass

import torch

from oxr_inference_b200 import ops
from oxr_inference_b200.cache.manager import RequestCache, pages_for
from oxr_inference_b200.engine.runtime import no_collection
from oxr_inference_b200.parts.base import StepContext

CHUNK = 64
"""Steps whose tokens are kept on the GPU before the host reads them."""
LOOPS = 8
"""Graphs that are kept: one for each number of requests and width of their tables, the ones used last."""


@dataclass
class _Loop:
    """What one graph reads and writes, for so many requests and pages of a table's row."""

    tokens: torch.Tensor        # int32 [requests]: each request's next token
    state_slots: torch.Tensor   # int32 [requests]
    ones: torch.Tensor
    rows: torch.Tensor          # 0, 1, ...
    nothing: torch.Tensor       # -1
    zeros: torch.Tensor
    groups: list[tuple[torch.Tensor, ...]]   # per group: lengths, held pages, block table, free list and its count
    out: torch.Tensor           # int32 [CHUNK, requests]
    turn: torch.Tensor          # int64 [1]: the row of ``out`` that the next step fills
    graph: torch.cuda.CUDAGraph | None = None
    kernels: int = 0


class DeviceDecode:
    def __init__(self, runner):
        self.runner = weakref.proxy(runner)      # (which owns this: a circle would keep graphs and pools until garbage is collected)
        self._loops: dict[tuple[int, int], _Loop] = {}
        self._pool = None

    @torch.inference_mode()
    def run(self, requests: list[RequestCache], tokens: list[int], steps: int) -> list[list[int]]:
        """The next ``steps`` tokens of each request, greedily (the first largest logit), from ``tokens``: the last token each has, not yet in its cache.
        Afterwards each request's cache holds ``steps`` tokens more: the given one and all but the last of those returned. If a kernel reports an error
        (RuntimeError), the requests' lengths are as before, but their pages and states are not: they have to be closed."""
        m = self.runner.cache
        if not requests or len(requests) != len(tokens) or steps < 1:
            raise ValueError(f"{len(requests)} requests, {len(tokens)} tokens, {steps} steps")
        if len({id(rc) for rc in requests}) != len(requests):
            raise ValueError("a request is given twice")
        vocabulary = self.runner.model.spec.vocab_size
        if not all(0 <= t < vocabulary for t in tokens):
            raise ValueError(f"a token outside the vocabulary of {vocabulary}")
        if not m.pools:
            raise ValueError("the model keeps no pages; its steps need no tables")
        longest = max(rc.length for rc in requests) + steps
        if longest > self.runner.model.runtime.max_positions:
            raise ValueError(f"{longest} positions, the model has {self.runner.model.runtime.max_positions}")
        lacking = sum(max(0, pages_for(rc.length + steps, m.page_size) - pages_for(rc.room, m.page_size)) for rc in requests)
        if lacking > m.free_pages or not all(m.reserve(rc, rc.length + steps) for rc in requests):
            raise RuntimeError(f"the cache lacks pages for {steps} more tokens of {len(requests)} requests ({m.free_pages} free)")
        n, width = len(requests), 16
        while width < max(len(t) for rc in requests for t in rc.tables):
            width *= 2
        loop = self._loops.pop((n, width), None)
        if loop is None:
            while len(self._loops) >= LOOPS:      # (none is under way: each call waits for its own)
                del self._loops[next(iter(self._loops))]
            loop = self._capture(n, width)
        self._loops[(n, width)] = loop      # the last to go

        def put(dst: torch.Tensor, values: list) -> None:
            dst.copy_(torch.tensor(values, dtype=dst.dtype).view(dst.shape))

        put(loop.tokens, tokens)
        put(loop.state_slots, [rc.state_slot for rc in requests])
        for g, (lengths, held, table, _, _) in enumerate(loop.groups):
            fill = m.scratch_pages[g] if m.scratch_pages else 0
            put(lengths, [rc.length for rc in requests])
            put(held, [len(rc.tables[g]) for rc in requests])
            put(table, [rc.tables[g] + [fill] * (width - len(rc.tables[g])) for rc in requests])
        chosen: list[list[int]] = [[] for _ in requests]
        for first in range(0, steps, CHUNK):
            count = min(CHUNK, steps - first)
            loop.turn.zero_()
            for _ in range(count):
                loop.graph.replay()
            ops.launch_count += loop.kernels * count
            for out, column in zip(chosen, loop.out[:count].t().tolist()):
                out += column
            self.runner.check()
        for rc in requests:
            m.advance(rc, rc.length + steps)
        self.runner.steps += steps
        return chosen

    def _step(self, n: int, width: int, loop: _Loop) -> None:
        runner = self.runner
        m, status = runner.cache, runner.model.runtime.status
        views, first = [], None
        for g, (lengths, held, table, free_list, free_count) in enumerate(loop.groups):
            s = ops.step_pages(lengths, held, table, free_list, free_count, loop.ones, page_size=m.page_size, tokens=n, status=status, advance=True)
            first = first or s
            views.append(m.group_view(g, table, s.slots))
        ctx = StepContext(
            n_tokens=n, n_requests=n, token_ids=loop.tokens, positions=first.positions, req_of_token=first.req_of_token, cu_q=first.cu_q,
            ctx_lens=first.ctx_lens, state_slots=loop.state_slots, logit_rows=loop.rows, no_store_slots=loop.nothing, groups=views,
            tiles={spec: (loop.rows, loop.zeros, n if spec[1] <= 1 else 0) for spec in runner.builder.tile_specs},
            kv_len_bound=width * m.page_size, q_lens=[1] * n, ctx_lens_host=[1] * n, status=status)
        tokens = ops.sample(runner.model.step(ctx, m))
        loop.tokens.copy_(tokens)
        loop.out.index_copy_(0, loop.turn, tokens[None])
        loop.turn.add_(1)

    def _capture(self, n: int, width: int) -> _Loop:
        m = self.runner.cache
        dev = self.runner.model.runtime.device

        def ints(value: int, *shape: int) -> torch.Tensor:
            return torch.full(shape, value, dtype=torch.int32, device=dev)

        groups = [(ints(0, n), ints(1, n), ints(m.scratch_pages[g] if m.scratch_pages else 0, n, width), ints(0, 1), ints(0, 1)) for g in range(len(m.pools))]
        loop = _Loop(ints(0, n), ints(m.scratch_slot, n), ints(1, n), torch.arange(n, dtype=torch.int32, device=dev), ints(-1, n), ints(0, n), groups,
                     ints(0, CHUNK, n), torch.zeros(1, dtype=torch.int64, device=dev))
        # One eager step first, of rows that read and write the scratch page and the scratch state alone, so that what is set up at a first call
        # is set up outside the capture.
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self._step(n, width, loop)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        if self._pool is None:
            self._pool = torch.cuda.graph_pool_handle()
        before = ops.launch_count
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), no_collection():
            graph.capture_begin(pool=self._pool)
            try:
                self._step(n, width, loop)
            finally:
                graph.capture_end()
        torch.cuda.current_stream().wait_stream(side)
        loop.kernels, ops.launch_count = ops.launch_count - before, before    # capturing launches nothing
        loop.graph = graph
        return loop
