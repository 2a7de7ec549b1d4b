"""Entry points of the kernels around the 8-bit paged cache: the store that fills it, attention over it, and a step's page tables on the GPU.

The cache holds e4m3 codes: one layer's pools are ``[pages, page_size, KV, D]`` of ``torch.float8_e4m3fn`` with fp32 scales ``[pages, KV]``; an
entry is its code times the scale of its page and KV head. Zeroed scales make an empty cache. The reference keeps keys and values in the model's
16-bit type only (oxr_runtime/kv_cache.py:27-29); the masking rule is that of its ``paged_extend`` (oxr_runtime/attention.py:96-109). ``step_pages``
does on the GPU what the reference's host does between two steps (oxr_runtime/kv_cache.py:43-72, oxr_runtime/language.py:320-322).
"""

from __future__ import annotations

import functools
import struct
from ctypes import c_char_p, c_int
from typing import NamedTuple

import torch

from oxr_inference_b200 import ops
from oxr_inference_b200.ops import build
from oxr_inference_b200.ops.build import BuildError

KV8_DTYPE = torch.float8_e4m3fn
KV8_FEW_TOKENS = 1024
"""Up to so many tokens the store looks through all slots itself; for more it takes scratch of two words a page."""
KV8_LONGEST_PAGE = 8192
"""Tokens of a page that the store takes at most."""
_INT, _F32 = torch.int32, torch.float32

# The calls' arguments, each in one block as the libraries declare it: pointers first, then 64-bit and 32-bit numbers.
_ATTENTION_CALL = struct.Struct("@12Q2q14if").pack
_STORE_CALL = struct.Struct("@10Q3q6i").pack
_PAGES_CALL = struct.Struct("@14Q6i").pack

_kv8: dict = {}
_core = None


def _kv8_lib(head_dim: int):
    lib = _kv8.get(head_dim)
    if lib is None:
        lib = build.kv8_library(head_dim)
        lib.oxr_kv8_attention.argtypes = [c_char_p]
        lib.oxr_kv8_attention.restype = c_int
        lib.oxr_kv8_prompt_attention.argtypes = [c_char_p]
        lib.oxr_kv8_prompt_attention.restype = c_int
        lib.oxr_kv8_prompt_ready.restype = c_int
        lib.oxr_kv8_blocks_per_sm.argtypes = [c_int, c_int]
        lib.oxr_kv8_blocks_per_sm.restype = c_int
        lib.oxr_kv8_head_dim.restype = c_int
        if lib.oxr_kv8_head_dim() != head_dim:
            raise BuildError(f"library for head size {head_dim} reports {lib.oxr_kv8_head_dim()}")
        lib.oxr_set_chain.argtypes = [c_int]
        lib.oxr_set_chain.restype = None
        lib.oxr_set_chain(int(ops.CHAIN_KERNELS))
        _kv8[head_dim] = lib
    return lib


def _core_lib():
    global _core
    if _core is None:
        lib = ops._lib()
        lib.oxr_store_kv8.argtypes = [c_char_p]
        lib.oxr_store_kv8.restype = c_int
        lib.oxr_step_pages.argtypes = [c_char_p]
        lib.oxr_step_pages.restype = c_int
        lib.oxr_store_kv8_few.restype = c_int
        if lib.oxr_store_kv8_few() != KV8_FEW_TOKENS:
            raise BuildError(f"the store's kernels take up to {lib.oxr_store_kv8_few()} tokens without scratch, the host {KV8_FEW_TOKENS}")
        _core = lib
    return _core


def warm_up_kv8(head_dims: tuple[int, ...]) -> None:
    """Build and load the libraries of an 8-bit cache with these head sizes, before the first step."""
    if head_dims:
        _core_lib()
    for d in head_dims:
        _kv8_lib(d)


def _here(t: torch.Tensor, name: str) -> None:
    """The launch goes to the current device's current stream, so the tensors have to be there."""
    if not t.is_cuda:
        raise ops.KernelError(f"{name} is on {t.device}; the kernels run on a CUDA device only (there is no CPU path)")
    if t.get_device() != ops._raw_device():
        raise ops.KernelError(f"{name} is on {t.device}, the current device is cuda:{ops._raw_device()}")


# The checks are laid out for calls that pass them: a few comparisons in one expression each, and a function that finds the words for one that does not.
# (Outside of CUDA graphs a small step's calls are bound by the host: attention 17.7 us a call instead of 23, tables 14 instead of 19, the store 9.2 instead of 11.5.)
def _plain(t: torch.Tensor, device: int, dtype: torch.dtype) -> bool:
    return t.dtype is dtype and t.is_contiguous() and t.get_device() == device


def _refuse_plain(device: int, dtype: torch.dtype, **tensors: torch.Tensor) -> None:
    for name, t in tensors.items():
        if not _plain(t, device, dtype):
            raise ops.KernelError(f"{name} must be contiguous {dtype} on cuda:{device}, got {t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}")


def _need_pools(device: int, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(pages, page size, KV heads, head size, bytes from page to page) of the pools, which may be slices of wider ones as long as each page is whole."""
    shape, strides = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or k_cache.dtype is not KV8_DTYPE or v_cache.dtype is not KV8_DTYPE or v_cache.shape != shape:
        raise ops.KernelError(f"the pools must be [pages, page size, KV heads, head size] of {KV8_DTYPE}, got {k_cache.dtype} {tuple(shape)} and "
                              f"{v_cache.dtype} {tuple(v_cache.shape)}")
    pages, page, kv, d = shape
    if not (pages and page and kv and d):
        raise ops.KernelError(f"pools of {tuple(shape)}: there is nothing in them")
    row = kv * d
    if max(pages, page, row) > 0x7fffffff:
        raise ops.KernelError(f"pools of {tuple(shape)}: pages, their tokens and the bytes of a token are counted in 32 bits")
    stride = strides[0]
    if (strides != (stride, row, d, 1) or v_cache.stride() != strides or stride < page * row or (stride | d | k_cache.data_ptr() | v_cache.data_ptr()) % 16
            or k_cache.get_device() != device or v_cache.get_device() != device):
        raise ops.KernelError(f"pools with strides {strides} and {v_cache.stride()}: pages must be whole, 16-byte aligned and as far apart in both, "
                              f"head sizes multiples of 16, on cuda:{device}")
    if not (k_scale.dtype is v_scale.dtype is _F32 and k_scale.is_contiguous() and v_scale.is_contiguous() and k_scale.get_device() == v_scale.get_device() == device):
        _refuse_plain(device, _F32, k_scale=k_scale, v_scale=v_scale)
    if k_scale.shape != (pages, kv) or v_scale.shape != (pages, kv):
        raise ops.KernelError(f"one scale per page and KV head: {tuple(k_scale.shape)}, {tuple(v_scale.shape)} for pools of {pages} pages and {kv} heads")
    return pages, page, kv, d, stride


def _head_rows(t: torch.Tensor, name: str, device: int) -> int:
    """Entries from token to token of ``[tokens, heads, size]``; tokens may lie apart, their rows 16-byte aligned."""
    if t.get_device() != device:
        raise ops.KernelError(f"{name} is on {t.device}, not on cuda:{device}")
    if t.is_contiguous():
        stride = t.shape[1] * t.shape[2]
    else:
        stride, head, one = t.stride()
        if one != 1 or head != t.shape[2] or stride < t.shape[1] * t.shape[2]:
            raise ops.KernelError(f"{name}: {t.dtype} {tuple(t.shape)} with strides {t.stride()}: a token's heads must lie side by side")
    if t.data_ptr() % 16 or stride * t.element_size() % 16:
        raise ops.KernelError(f"{name}: rows must be 16-byte aligned")
    return stride


def store_kv8(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
              v_scale: torch.Tensor, status: torch.Tensor) -> None:
    """New keys and values ``[n, KV, D]`` (float32 or bfloat16, tokens may lie apart) into the 8-bit pools at ``slots`` (int32, page * page size +
    place; a negative one skips its token), in any order; of two tokens with one slot the later stays.

    A page's scale is a power of two, one for each KV head and for keys and values apart: the least 2^e whose 448-fold reaches every magnitude stored since
    the page was begun. Storing a page's first slot begins it (what its other slots held is void); after that the scale only grows, and what the
    page holds is then rounded to the new scale (exact but for codes below e4m3's normal range). Infinities and NaN become NaN and have no say in
    the scale. A slot outside the pool sets the status word and is skipped. Measured on a B200 (8 KV heads of 128): 64 tokens 3.3 us, 10,300 tokens 22 us."""
    _here(k_cache, "k_cache")
    device = k_cache.get_device()
    pages, page, kv, d, page_stride = _need_pools(device, k_cache, v_cache, k_scale, v_scale)
    n = slots.shape[0]
    if not (_plain(slots, device, _INT) and _plain(status, device, _INT)):
        _refuse_plain(device, _INT, slots=slots, status=status)
    if slots.dim() != 1 or k.shape != (n, kv, d) or v.shape != (n, kv, d) or k.dtype != v.dtype:
        raise ops.KernelError(f"k {k.dtype} {tuple(k.shape)} and v {v.dtype} {tuple(v.shape)} must be [{n}, {kv}, {d}] of one dtype for {n} slots")
    code = ops._dtype_code(k)
    if page > KV8_LONGEST_PAGE or pages * page > 0x80000000 - KV8_LONGEST_PAGE:
        raise ops.KernelError(f"{pages} pages of {page} tokens: the store takes pages of up to {KV8_LONGEST_PAGE}, slots below 2^31 - {KV8_LONGEST_PAGE}")
    k_stride, v_stride = _head_rows(k, "k", device), _head_rows(v, "v", device)
    if n == 0:
        return
    ends = None if n <= KV8_FEW_TOKENS else slots.new_empty(2 * pages)
    call = _STORE_CALL(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k.data_ptr(), v.data_ptr(), slots.data_ptr(),
                       0 if ends is None else ends.data_ptr(), status.data_ptr(), ops._stream(), k_stride, v_stride, page_stride, n, pages, page, kv, d, code)
    ops._done(_core_lib().oxr_store_kv8(call), "store_kv8")
    if ends is not None:
        ops.launch_count += 1


@functools.lru_cache(maxsize=4096)
def _split_plan(requests: int, tokens: int, longest: int, group: int, kv: int, head_dim: int, code: int, seen: int) -> tuple[int, int, int]:
    """(rows of a tile, blocks, words of scratch) of the split-key kernel for portions of up to ``longest`` tokens; a tile's rows are (token, query head) pairs of
    one KV head."""
    rows = 8 if group * longest <= 8 else 16
    heads_per_tile = min(group, rows)
    per_tile = rows // heads_per_tile
    tiles = min(tokens, requests * -(-longest // per_tile), requests + tokens // per_tile) * kv * -(-group // heads_per_tile)
    blocks = kv8_blocks(tiles, -(-seen // 32), _kv8_room(head_dim, code, rows))
    return rows, blocks, 8 * blocks * rows * (head_dim + 3) + 32 * blocks


@functools.lru_cache(maxsize=None)
def _kv8_room(head_dim: int, code: int, tile_rows: int) -> int:
    """Blocks of the split-key kernel that the current device holds at a time."""
    return ops.num_sms() * _kv8_lib(head_dim).oxr_kv8_blocks_per_sm(code, tile_rows)


def kv8_blocks(tiles: int, key_blocks: int, room: int) -> int:
    """Blocks of four warps among which a step's work is dealt out: as many as the device holds at a time, fewer where a warp would get
    less than one block of 32 keys (``tiles`` tiles of at most ``key_blocks`` of them)."""
    return max(1, min(room, -(-tiles * key_blocks // 4)))


KV8_PROMPT_ROWS = 256
"""Rows of a tile of the tcgen05 kernel for long portions."""


@functools.lru_cache(maxsize=None)
def kv8_prompt_runs(head_dim: int) -> bool:
    """Whether this build of the tcgen05 kernel can run: its split of the registers is for 128 a thread, which is the compiler's choice."""
    return bool(_kv8_lib(head_dim).oxr_kv8_prompt_ready())


def kv8_prompt_takes(max_q_len: int, head_dim: int, dtype: torch.dtype, scale: float) -> bool:
    """Whether the tcgen05 kernel can take the longer portions of a step: bfloat16 queries, head sizes up to 128, a positive scale (it scales a row's maximum,
    not each score)."""
    return dtype == torch.bfloat16 and head_dim <= 128 and scale > 0 and max_q_len > ops.SHORT_MAX_TOKENS


def kv8_prompt_pays(requests: int, tokens: int, max_q_len: int, num_heads: int, num_kv_heads: int, head_dim: int, seen: int) -> bool:
    """Whether it is also the faster one for portions of more than ``ops.SHORT_MAX_TOKENS`` tokens that see up to ``seen`` keys. Its tiles (256 rows) walk over their
    keys alone, 2.5 us for each 128 of them, so that a few tiles leave most of the GPU idle; the split-key kernel deals all work out evenly but
    needs 1.8 ns for each 16 rows x 32 keys x 128 entries. Measured on a B200 (32 / 8 heads of 128), this one against that one: 64 tokens on 4,096 keys 87
    and 49 us, 128 on 8,192 160 and 125, 256 on 4,096 88 and 129, 512 on 512 24 and 52, 16 requests of 16 tokens on 2,048 51 and 76, 2,048 on 4,096 142 and 890."""
    group = num_heads // num_kv_heads

    def cut(rows: int) -> tuple[int, int]:      # tokens of a tile, tiles that the heads of all KV heads make
        heads = min(group, rows)
        return rows // heads, num_kv_heads * -(-group // heads)

    per_tile, across = cut(KV8_PROMPT_ROWS)
    tiles = max(-(-max_q_len // per_tile), tokens // per_tile, requests if tokens > ops.SHORT_MAX_TOKENS * requests else 1) * across
    short_per_tile, short_across = cut(16)
    items = tokens / short_per_tile * short_across * -(-seen // 32) * head_dim / 128
    return 15 + 2.5 * -(-seen // 128) * max(1.0, tiles / 148) < 12 + 0.0018 * items


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory from the first to the last entry of two tensors has bytes in common."""
    ends = [(t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()) for t in (a, b) if t.numel()]
    return len(ends) == 2 and max(ends[0][0], ends[1][0]) < min(ends[0][1], ends[1][1])


def paged_attention_kv8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, *,
                        cu_q: torch.Tensor, ctx_lens: torch.Tensor, block_table: torch.Tensor, scale: float, window: int = 0, max_q_len: int,
                        kv_len_bound: int, status: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal grouped-query attention of a step's new tokens over the 8-bit paged cache, which holds their keys and values already.

    ``q`` is ``[tokens, H, D]`` (float32 or bfloat16; tokens may lie apart), request r's new tokens are its rows ``cu_q[r] .. cu_q[r + 1] - 1`` at the
    last positions of its ``ctx_lens[r]`` cached ones; ``block_table`` ``[requests, pages]`` names its pages. With ``window`` > 0 a query sees its last
    ``window`` keys. A request may bring no token; a row that sees no key is zero; rows of ``out`` behind ``cu_q[-1]`` are left as they were.
    ``max_q_len``: no request brings more new tokens (one that does sets the status word and is left out); ``kv_len_bound``: about the longest context,
    which only decides how the keys are cut. No host list of tiles is needed, so the lengths may live on the GPU alone (see :func:`step_pages`).
    Scores, sums and softmax are fp32; weights, times the value scale of their key, are rounded to 11 bits for bfloat16 queries, to 22 for float32 ones. Those of
    less than 2^-17 of a row's largest (2^-29 in the kernel for few tokens) lose bits. Scales may be any numbers, zero, negative ones and NaN among them; those
    that :func:`store_kv8` makes (powers of two) are the fast ones while the value scales of neighbouring pages lie within 2^4 of each other."""
    _here(q, "q")
    device = q.get_device()
    pages, page, kv, d, page_stride = _need_pools(device, k_cache, v_cache, k_scale, v_scale)
    code = ops._dtype_code(q)
    if q.dim() != 3 or q.shape[2] != d or q.shape[1] % kv or q.shape[1] == 0:
        raise ops.KernelError(f"q {tuple(q.shape)} does not fit {kv} KV heads of {d}")
    tokens, heads = q.shape[0], q.shape[1]
    q_stride = _head_rows(q, "q", device)
    if not (cu_q.dtype is ctx_lens.dtype is block_table.dtype is status.dtype is _INT and cu_q.is_contiguous() and ctx_lens.is_contiguous()
            and block_table.is_contiguous() and status.is_contiguous()
            and cu_q.get_device() == ctx_lens.get_device() == block_table.get_device() == status.get_device() == device):
        _refuse_plain(device, _INT, cu_q=cu_q, ctx_lens=ctx_lens, block_table=block_table, status=status)
    n = ctx_lens.shape[0]
    if ctx_lens.dim() != 1 or cu_q.shape != (n + 1,) or block_table.dim() != 2 or block_table.shape[0] != n:
        raise ops.KernelError(f"cu_q {tuple(cu_q.shape)}, ctx_lens {tuple(ctx_lens.shape)} and block_table {tuple(block_table.shape)} are not of one batch")
    if window < 0 or max_q_len < 1:
        raise ops.KernelError(f"window {window}, max_q_len {max_q_len}")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((tokens, heads, d))
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.get_device() != device or out.data_ptr() % 16:
        raise ops.KernelError(f"out {out.dtype} {tuple(out.shape)} must be a contiguous tensor like q {q.dtype} {tuple(q.shape)}")
    elif out.untyped_storage().data_ptr() == q.untyped_storage().data_ptr() and _overlap(out, q):
        raise ops.KernelError("out lies over q, which is read more than once")
    if n == 0 or tokens == 0:
        return out
    lib = _kv8_lib(d)
    group = heads // kv
    longest = max_q_len = min(int(max_q_len), tokens)
    window = min(int(window), 1 << 30)      # more than any position: no window
    stream = ops._stream()
    pointers = (out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), cu_q.data_ptr(), ctx_lens.data_ptr(),
                block_table.data_ptr())
    sizes = (page_stride, q_stride, n, tokens, block_table.shape[1], page, pages, heads, kv, window)
    seen = max(1, min(kv_len_bound, window + max_q_len) if window > 0 else kv_len_bound)
    if max_q_len > ops.SHORT_MAX_TOKENS and kv8_prompt_takes(max_q_len, d, q.dtype, scale) and kv8_prompt_pays(n, tokens, max_q_len, heads, kv, d, seen) and kv8_prompt_runs(d):
        fewest = ops.SHORT_MAX_TOKENS + 1 if n > 1 else 1      # a request alone goes there whatever it brings
        tiles = min(tokens, min(n, tokens // fewest) + tokens // (KV8_PROMPT_ROWS // min(group, KV8_PROMPT_ROWS)))
        call = _ATTENTION_CALL(*pointers, 0, status.data_ptr(), stream, *sizes, fewest, max_q_len, max_q_len, 0, tiles, code, scale)
        ops._done(lib.oxr_kv8_prompt_attention(call), "paged_attention_kv8 (prompts)")
        longest = fewest - 1
        if longest == 0:
            return out
    seen = max(1, min(kv_len_bound, window + longest + 32) if window > 0 else kv_len_bound)
    rows, blocks, words = _split_plan(n, tokens, longest, group, kv, d, code, seen)
    scratch = k_scale.new_empty(words)
    call = _ATTENTION_CALL(*pointers, scratch.data_ptr(), status.data_ptr(), stream, *sizes, 1, longest, max_q_len, rows, blocks, code, scale)
    ops._done(lib.oxr_kv8_attention(call), "paged_attention_kv8")
    ops.launch_count += 1
    return out


class PageStep(NamedTuple):
    """What a step's kernels read, as :func:`step_pages` lays it out (int32 on the GPU)."""

    slots: torch.Tensor
    """``[tokens]`` cache slot of each new token; -1 behind the last one."""
    positions: torch.Tensor
    """``[tokens]`` position of each new token in its request; 0 behind the last one."""
    req_of_token: torch.Tensor
    """``[tokens]`` row of each new token's request; -1 behind the last one."""
    cu_q: torch.Tensor
    """``[rows + 1]`` each row's first new token."""
    ctx_lens: torch.Tensor
    """``[rows]`` each row's length with its new tokens."""


def step_pages(lengths: torch.Tensor, held: torch.Tensor, block_table: torch.Tensor, free_list: torch.Tensor, free_count: torch.Tensor, q_lens: torch.Tensor,
               fresh: torch.Tensor | None = None, *, page_size: int, tokens: int, status: torch.Tensor, advance: bool = False) -> PageStep:
    """Pages, block tables and slot maps of a step, worked out on the GPU from the lengths of its requests; nothing comes to the host, so it can stand in a
    CUDA graph with the layers that read it.

    Row r of ``block_table`` ``[rows, width]`` is a request with ``lengths[r]`` cached tokens on its first ``held[r]`` entries; ``q_lens[r]`` more are
    to come. Rows with ``fresh[r]`` other than 0 begin anew at length 0: their pages go on top of the stack ``free_list[:free_count[0]]``, row after row
    and page after page. Then every row takes the pages it lacks from the top, in the same order. A row that is given up is one with ``fresh`` 1 and
    ``q_lens`` 0. ``held``, ``block_table``, ``free_list`` and ``free_count`` are updated in place; with ``advance`` so is ``lengths`` (the step's tokens then count
    as cached), without it ``lengths`` stays as it was, and a step of rows that go on may be asked for again: it takes nothing more and says the same. A row that
    begins anew does so each time it is asked for: its pages go back and come again in another order. To ask for such a step again, set the row's length
    and ``fresh`` to 0 first.

    All or nothing: if pages are lacking, a row does not fit its numbers (longer than ``width`` pages, a negative length) or the step brings more than
    ``tokens`` tokens, the status word is set, nothing moves, and the arrays hold no token at all (slots -1, ``cu_q`` and ``ctx_lens`` 0). The numbers of
    pages are taken as they stand: a token on a negative one gets slot -1, on one beyond all pools a slot that the store reports."""
    _here(block_table, "block_table")
    device = block_table.get_device()
    if not (lengths.dtype is held.dtype is block_table.dtype is free_list.dtype is free_count.dtype is q_lens.dtype is status.dtype is _INT
            and lengths.is_contiguous() and held.is_contiguous() and block_table.is_contiguous() and free_list.is_contiguous() and free_count.is_contiguous()
            and q_lens.is_contiguous() and status.is_contiguous()
            and lengths.get_device() == held.get_device() == free_list.get_device() == free_count.get_device() == q_lens.get_device() == status.get_device() == device):
        _refuse_plain(device, _INT, lengths=lengths, held=held, block_table=block_table, free_list=free_list, free_count=free_count, q_lens=q_lens, status=status)
    if block_table.dim() != 2:
        raise ops.KernelError(f"block_table must be [rows, pages], got {tuple(block_table.shape)}")
    rows, width = block_table.shape
    one = (rows,)
    if lengths.shape != one or held.shape != one or q_lens.shape != one or fresh is not None and not (fresh.shape == one and _plain(fresh, device, _INT)):
        for name, t in (("lengths", lengths), ("held", held), ("q_lens", q_lens), ("fresh", fresh)):
            if t is not None and t.shape != one:
                raise ops.KernelError(f"{name} {tuple(t.shape)}: one for each of {rows} rows")
        _refuse_plain(device, _INT, fresh=fresh)
    if free_count.numel() != 1 or free_list.dim() != 1:
        raise ops.KernelError(f"free_list {tuple(free_list.shape)} must be a row and free_count {tuple(free_count.shape)} one number")
    if page_size < 1 or tokens < 0 or rows > 8192 or max(width, free_list.shape[0], 1) * page_size > 0x7fffffff or 3 * tokens > 0x7fffffff:
        raise ops.KernelError(f"page size {page_size}, {tokens} tokens, {rows} rows of {width} pages, {free_list.shape[0]} in all: at most 8192 rows, positions and slots below 2^31")
    block = block_table.new_empty(3 * tokens + 2 * rows + 1)
    step = PageStep(*torch.split_with_sizes(block, (tokens, tokens, tokens, rows + 1, rows)))
    at = block.data_ptr()
    call = _PAGES_CALL(lengths.data_ptr(), held.data_ptr(), block_table.data_ptr(), free_list.data_ptr(), free_count.data_ptr(), q_lens.data_ptr(),
                       0 if fresh is None else fresh.data_ptr(), at, at + 4 * tokens, at + 8 * tokens, at + 12 * tokens, at + 4 * (3 * tokens + rows + 1),
                       status.data_ptr(), ops._stream(), rows, width, page_size, free_list.shape[0], tokens, 1 if advance else 0)
    ops._done(_core_lib().oxr_step_pages(call), "step_pages")
    return step
