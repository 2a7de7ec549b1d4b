"""The 8-bit paged cache in plain 64-bit arithmetic: its store, attention over it, and page tables with Python lists."""

from __future__ import annotations

import math

import torch

LARGEST = 448.0


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number (ties to even), in 64 bits; NaN for what is not finite."""
    x = x.double()
    finite = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    _, exponent = torch.frexp(finite)
    step = torch.ldexp(torch.ones_like(finite), (exponent - 4).clamp(min=-9))
    out = (torch.round(finite / step) * step).clamp(-LARGEST, LARGEST)
    return torch.where(torch.isfinite(x), out, torch.full_like(out, math.nan))


def scale_for(most: float) -> float:
    """The least power of two (from 2^-118 on) whose 448-fold reaches ``most``."""
    if most == 0:
        return 0.0
    e = -118
    while LARGEST * 2.0 ** e < most:
        e += 1
    return 2.0 ** e


def store(x: torch.Tensor, slots: list[int], codes: torch.Tensor, scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [n, KV, D]`` into ``codes [pages, page, KV, D]`` / ``scales [pages, KV]``: new codes and scales in 64 bits."""
    codes, scales, x = codes.double().clone(), scales.double().clone(), x.double()
    page = codes.shape[1]
    where: dict[int, dict[int, int]] = {}
    for t, s in enumerate(slots):
        if 0 <= s < codes.shape[0] * page:
            where.setdefault(s // page, {})[s % page] = t    # the later token stays
    for p, tokens in where.items():
        for h in range(codes.shape[2]):
            new = x[list(tokens.values()), h]
            finite = new[torch.isfinite(new)].abs()
            need = scale_for(float(finite.max()) if finite.numel() else 0.0)
            old = 0.0 if 0 in tokens else float(scales[p, h])
            scale = max(old, need)
            if 0 not in tokens and scale > old:
                kept = [o for o in range(page) if o not in tokens]
                codes[p, kept, h] = e4m3(codes[p, kept, h] * (old / scale))
            codes[p, list(tokens), h] = e4m3(new / scale if scale else new * 0)
            scales[p, h] = scale
    return codes, scales


def attention(q, k_codes, v_codes, k_scale, v_scale, q_lens, ctx_lens, tables, scale, window=0):
    """Output, sum of weights times |values| and the largest sum of |q||k| |scale| of each row, in 64 bits. Keys that a row does not see have no part in it."""
    n, heads, d = q.shape
    page, kv = k_codes.shape[1], k_codes.shape[2]
    out = torch.zeros((n, heads, d), dtype=torch.float64)
    spread, size = torch.zeros_like(out), torch.zeros((n, heads, 1), dtype=torch.float64)
    q, kc, vc, ks, vs = (x.double().cpu() for x in (q, k_codes, v_codes, k_scale, v_scale))
    at = 0
    for r, (ql, ctx) in enumerate(zip(q_lens, ctx_lens)):
        keys = torch.arange(max(ctx, 0))
        pages = torch.tensor(tables[r], dtype=torch.long)[keys // page] if ctx > 0 else keys
        k = kc[pages, keys % page] * ks[pages][:, :, None]
        v = vc[pages, keys % page] * vs[pages][:, :, None]
        for i in range(ql):
            pos = ctx - ql + i
            lo = max(0, pos - window + 1) if window else 0
            if pos < 0:
                at += 1
                continue
            for h in range(heads):
                g = h // (heads // kv)
                kk, vv = k[lo:pos + 1, g], v[lo:pos + 1, g]
                w = torch.softmax(kk @ q[at, h] * scale, 0)
                out[at, h], spread[at, h] = w @ vv, w @ vv.abs()
                size[at, h] = (kk.abs() @ q[at, h].abs()).max() * abs(scale)
            at += 1
    return out, spread, size


def tolerance(out, spread, size, dtype, head_dim, keys):
    """How far a kernel may be off. The result is rounded to its type; weights are rounded to one fp16 number (bf16 queries) or two of
    them (fp32): an fp16 number has 11 significant bits, half a step is 2^-11 of a number just above a power of two, and the second number leaves 2^-11 of that; they come from an exp2 good to
    2^-22 twice (numerator and denominator); a score's fp32 sum of ``head_dim`` products and its two factors err by 2^-22 of the sum of their
    magnitudes each at most (the tensor cores cut instead of rounding), which moves a weight by as much; and the sum over the keys, 16 at a time, errs in the same way."""
    half = torch.finfo(dtype).eps / 2
    weight = 2.0 ** (-11 if dtype == torch.bfloat16 else -22) + 2 * 2.0 ** -22 + 2 * (head_dim / 16 + 8) * 2.0 ** -22 * size + (keys / 16 + 20) * 2.0 ** -22
    return half * out.abs() + weight * spread * 1.01 + 1e-37


def pages(lengths, held, table, free, q_lens, fresh, page):
    """A step's tables with lists: (held, table, the whole stack with what lies above its top, count, begin, boundaries). ``free``: (list, count)."""
    held, table, (stack, count) = list(held), [list(r) for r in table], (list(free[0]), free[1])
    begin = list(lengths)
    for r, f in enumerate(fresh):
        if f:
            for j in range(held[r]):
                stack[count] = table[r][j]
                count += 1
            held[r] = begin[r] = 0
    cu = [0]
    for r, q in enumerate(q_lens):
        want = max(held[r], -(-(begin[r] + q) // page))
        while held[r] < want:
            count -= 1
            table[r][held[r]] = stack[count]
            held[r] += 1
        cu.append(cu[-1] + q)
    return held, table, stack, count, begin, cu
