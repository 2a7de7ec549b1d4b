"""The operators of the 8-bit paged cache whose speed is watched: what fills it, what reads it, and the page tables both go by.

A case's ``op`` is one of

* ``store``: new keys and values are rounded to e4m3 and put at their slots; every page has one scale for each KV head, a power of two that only
  grows while the page fills, so that what the page holds already is rounded again when a larger entry arrives;
* ``attention``: causal grouped-query attention of a step's new tokens over such a cache;
* ``pages``: block tables, cache slots, positions and boundaries of a step, worked out on the GPU from the lengths of its requests: rows that start
  anew give their pages back, then every row takes the pages that its new tokens need from the free list;
* ``step``: the three in a row, as one layer of a decode step has them.

Fields: ``requests``; ``context``: the longest context before the step, ``spread``: whether contexts are spread from one token up to it over their
logarithm or all alike; ``new``: the most new tokens of a request (with 1 each brings exactly one, else between one and that); ``heads``,
``kv_heads``, ``dim``, ``page`` (tokens), ``window`` (0: none), ``dtype`` (of queries, keys and values as they come); ``width``: pages that a
row of the block table has room for; ``fresh``: one row in so many starts anew (0: none).
"""

import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
LARGEST = 448.0          # of e4m3
SMALLEST_SCALE = -118    # binary exponent


def _case(name, op, **fields):
    out = {} if name is None else {"name": name}
    out.update(op=op, **fields)
    return out


def listed():
    qwen = dict(heads=32, kv_heads=8, dim=128, page=16, window=0, dtype="bfloat16")   # an attention layer of the 8B Qwen3 model
    return [
        # the decode step's store: 64 requests, one token each, somewhere inside their last page
        _case("store_decode_64", "store", requests=64, context=2048, new=1, kv_heads=8, dim=128, page=16, dtype="bfloat16"),
        # a full step of prompt portions
        _case("store_prompts", "store", requests=5, context=500, new=3277, kv_heads=8, dim=128, page=16, dtype="bfloat16"),
        # a true 32-bit engine with an odd page and head size: a few tokens of each request
        _case("store_fp32_odd", "store", requests=9, context=700, new=7, kv_heads=3, dim=80, page=24, dtype="float32"),
        # one user alone: the latency of a decode step
        _case("attention_decode_1", "attention", requests=1, context=2048, spread=False, new=1, **qwen),
        # the benchmark's largest decode batch
        _case("attention_decode_64", "attention", requests=64, context=2048, spread=False, new=1, **qwen),
        # a busy server whose requests differ in length by orders of magnitude
        _case("attention_decode_ragged", "attention", requests=24, context=32768, spread=True, new=1, **qwen),
        # the second portion of a long prompt
        _case("attention_prompt", "attention", requests=1, context=2048, spread=False, new=2048, **qwen),
        # short continuations and portions behind a window, all query heads on two KV heads
        _case("attention_window", "attention", requests=16, context=3000, spread=True, new=40, heads=16, kv_heads=2, dim=64, page=32, window=512, dtype="bfloat16"),
        # a trace replayed in true 32 bits, a few tokens of each request, an odd head size
        _case("attention_fp32", "attention", requests=5, context=3001, spread=True, new=8, heads=12, kv_heads=4, dim=80, page=16, window=1024, dtype="float32"),
        # continuous batching: 256 requests decode, one in 16 has just been replaced by a new one
        _case("pages_decode_256", "pages", requests=256, context=8192, new=1, page=16, width=2560, fresh=16),
        # prompts of ragged lengths arrive in all rows
        _case("pages_prompts", "pages", requests=48, context=4000, new=340, page=16, width=512, fresh=2),
        # one layer of a decode step: tables, store, attention
        _case("step_decode_32", "step", requests=32, context=1500, spread=True, new=1, width=128, fresh=0, **qwen),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("store", "attention", "attention", "attention", "pages", "step"))
    page = rng.choice((8, 16, 16, 16, 32, 64, 24))
    dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
    dim = rng.choice((128, 128, 64, 80, 48, 256))
    kv = rng.choice((1, 2, 3, 4, 8))
    group = rng.choice((1, 2, 4, 5, 8))
    if op == "pages":
        new = rng.choice((1, 1, _log(rng, 2, 200)))
        requests = _log(rng, 1, 512 if new == 1 else 40)
        return _case(None, op, requests=requests, context=_log(rng, 1, 8000), new=new, page=page, width=-(-8400 // page), fresh=rng.choice((0, 1, 2, 7)))
    if op == "store":
        new = rng.choice((1, 1, _log(rng, 2, 1500)))
        return _case(None, op, requests=_log(rng, 1, 200 if new == 1 else 8), context=_log(rng, 1, 2000), new=new, kv_heads=kv, dim=dim, page=page, dtype=dtype)
    new = 1 if op == "step" else rng.choice((1, 1, rng.randint(2, 8), _log(rng, 9, 700)))
    requests = _log(rng, 1, 40 if new <= 8 else 4)
    context = _log(rng, 1, min(16000, max(1, 60000 // requests)))
    window = rng.choice((0, 0, 0, rng.randint(1, 2000)))
    more = dict(width=-(-(context + 600) // page), fresh=rng.choice((0, 3))) if op == "step" else {}
    return _case(None, op, requests=requests, context=context, spread=rng.random() < 0.5, new=new, heads=kv * group, kv_heads=kv, dim=dim, page=page,
                 window=window, dtype=dtype, **more)


# ------------------------------------------------------------------------------------------------------------------------------ inputs
def _lengths(case, rng):
    """(contexts before the step, new tokens) of the requests."""
    n, most = case["requests"], case["context"]
    if case["op"] in ("store", "pages"):
        before = [rng.randint(0, most) for _ in range(n)]
    elif case["spread"]:
        before = [most] + [_log(rng, 1, most) for _ in range(n - 1)]
    else:
        before = [most] * n
    if case["new"] == 1 or (n == 1 and case["op"] == "attention"):
        new = [case["new"]] * n
    else:
        new = [rng.randint(max(1, case["new"] // 4), case["new"]) for _ in range(n)]
    return before, new


def _host_lengths(case):
    """The same for every seed, so that outputs have one shape."""
    return _lengths(case, random.Random(" ".join(str(case[k]) for k in sorted(case) if k != "name")))


def _anew(case):
    """Which rows start anew: one in so many."""
    return [int(case["fresh"] > 0 and i % case["fresh"] == case["fresh"] // 2) for i in range(case["requests"])]


def _quantised(x):
    """Codes and scales of whole pages ``[pages, page, heads, dim]``."""
    scale = _scale_for(x.abs().amax(dim=(1, 3)))
    inverse = torch.where(scale > 0, 1 / scale, torch.zeros_like(scale))
    return (x * inverse[:, None, :, None]).to(torch.float8_e4m3fn), scale


def _scale_for(largest):
    """The smallest power of two that brings ``largest`` into e4m3's range; 0 for 0."""
    mantissa, exponent = torch.frexp(largest)
    exponent = torch.where(mantissa <= LARGEST / 512, exponent - 9, exponent - 8).clamp(min=SMALLEST_SCALE)
    return torch.where(largest > 0, torch.ldexp(torch.ones_like(largest), exponent), torch.zeros_like(largest))


def _ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    before, new = _host_lengths(case)
    n, page, op = case["requests"], case["page"], case["op"]
    total = sum(new)
    s = {"op": op, "page": page, "total": total, "status": torch.zeros(4, dtype=torch.int32, device="cuda"), "q_lens": _ints(new)}
    held = [-(-b // page) for b in before]
    if op in ("pages", "step"):
        starts_anew = _anew(case)
        s["fresh"] = _ints(starts_anew)
        before_step = [0 if f else b for f, b in zip(starts_anew, before)]
        after = [max(h, -(-(b + q) // page)) for h, b, q in zip(held, before, new)]
        pool = sum(after) + n + 5
        table = torch.full((n, case["width"]), -1, dtype=torch.int32)
        order = random.Random(seed + 1).sample(range(pool), pool)
        at = 0
        for i, h in enumerate(held):
            table[i, :h] = torch.tensor(order[at:at + h], dtype=torch.int32)
            at += h
        free = torch.full((pool,), -1, dtype=torch.int32)
        free[:pool - at] = torch.tensor(order[at:], dtype=torch.int32)
        s.update(lengths=_ints(before), held=_ints(held), table=table.cuda(), free_list=free.cuda(), free_count=_ints([pool - at]))
        if op == "pages":
            return s
    else:
        before_step = before
        pages_of = [-(-(b + q) // page) for b, q in zip(before, new)]
        pool = sum(pages_of) + 3
        order = random.Random(seed + 1).sample(range(pool), pool)
        table = torch.full((n, max(pages_of)), -1, dtype=torch.int32)
        at = 0
        for i, h in enumerate(pages_of):
            table[i, :h] = torch.tensor(order[at:at + h], dtype=torch.int32)
            at += h
        s["table"] = table.cuda()
        cu = [0]
        for q in new:
            cu.append(cu[-1] + q)
        s.update(cu_q=_ints(cu), ctx_lens=_ints([b + q for b, q in zip(before, new)]))
        slots = []
        for i, (b, q) in enumerate(zip(before, new)):
            row = table[i].tolist()
            slots += [row[p // page] * page + p % page for p in range(b, b + q)]
        s["slots"] = _ints(slots)
    kv, dim, dtype = case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    # keys have channels that are larger than the others, and tokens differ in size; values less so
    channels = 1 + 6 * (torch.rand((kv, dim), generator=gen, device="cuda") < 0.04)

    def made(rows):
        k = torch.randn((rows, kv, dim), generator=gen, device="cuda") * channels
        v = torch.randn((rows, kv, dim), generator=gen, device="cuda") * torch.exp(0.5 * torch.randn((rows, 1, 1), generator=gen, device="cuda"))
        return k, v

    k, v = made(pool * page)
    s["k_cache"], s["k_scale"] = _quantised(k.view(pool, page, kv, dim))
    s["v_cache"], s["v_scale"] = _quantised(v.view(pool, page, kv, dim))
    del k, v
    if op in ("store", "step"):
        k, v = made(total)
        s["k"], s["v"] = k.to(dtype), v.to(dtype)
    if op in ("attention", "step"):
        s["q"] = torch.randn((total, case["heads"], dim), generator=gen, device="cuda").to(dtype)
        s.update(scale=dim ** -0.5, window=case["window"], most_new=max(new), longest=max(b + q for b, q in zip(before_step, new)))
    return s


# ------------------------------------------------------------------------------------------------------------------------------ the plain forms
def _store(cache, scales, x, slots, page):
    """One of the two pools: in place."""
    pages, offsets = (slots // page).long(), (slots % page).long()
    kv = x.shape[1]
    x = x.float()
    largest = torch.zeros_like(scales).scatter_reduce(0, pages[:, None].expand(-1, kv), x.abs().amax(-1), "amax")
    count = scales.shape[0]
    touched = torch.zeros(count, dtype=torch.bool, device=x.device).index_fill_(0, pages, True)
    begun = torch.zeros(count, dtype=torch.int32, device=x.device).scatter_reduce(0, pages, (offsets == 0).int(), "amax").bool()
    old = torch.where(begun[:, None], torch.zeros_like(scales), scales)
    scale = torch.where(touched[:, None], torch.maximum(old, _scale_for(largest)), scales)
    grown = touched[:, None] & ~begun[:, None] & (scale > old)
    ratio = torch.where(grown, old / scale, torch.ones_like(scale))
    cache.copy_((cache.float() * ratio[:, None, :, None]).to(cache.dtype))
    inverse = torch.where(scale > 0, 1 / scale, torch.zeros_like(scale))
    cache[pages, offsets] = (x * inverse[pages][:, :, None]).to(cache.dtype)
    scales.copy_(scale)


def _attention(q, k_cache, v_cache, k_scale, v_scale, cu_q, ctx_lens, table, scale, window, most_new, longest):
    tokens, heads, dim = q.shape
    page, kv = k_cache.shape[1], k_cache.shape[2]
    n, group = table.shape[0], heads // kv
    width = -(-longest // page)
    at = table[:, :width].long().clamp(min=0)

    def read(cache, scales):
        x = cache.view(torch.uint8)[at].view(cache.dtype).float() * scales[at][:, :, None, :, None]
        return x.reshape(n, width * page, kv, dim).permute(0, 2, 1, 3)

    new = cu_q[1:] - cu_q[:-1]
    token = torch.arange(tokens, device=q.device)
    req = torch.searchsorted(cu_q[1:].contiguous(), token, right=True)
    place = token - cu_q[req]
    padded = torch.zeros((n, most_new, heads, dim), device=q.device)
    padded[req, place] = q.float()
    rows = padded.view(n, most_new, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, most_new * group, dim)
    scores = torch.matmul(rows, read(k_cache, k_scale).transpose(2, 3)).view(n, kv, most_new, group, -1) * scale
    position = (ctx_lens - new)[:, None] + torch.arange(most_new, device=q.device)[None]
    key = torch.arange(width * page, device=q.device)
    seen = key[None, None] <= position[:, :, None]
    if window > 0:
        seen &= key[None, None] > position[:, :, None] - window
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    largest = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(largest > -math.inf, largest, torch.zeros_like(largest)))
    total = weights.sum(-1, keepdim=True)
    weights = weights / torch.where(total > 0, total, torch.ones_like(total))
    values = read(v_cache, v_scale)
    values = torch.where(key[None, None, :, None] < ctx_lens[:, None, None, None], values, torch.zeros_like(values))
    out = torch.matmul(weights.view(n, kv, most_new * group, -1), values).view(n, kv, most_new, group, dim)
    return out.permute(0, 2, 1, 3, 4).reshape(n, most_new, heads, dim)[req, place].to(q.dtype)


def _pages(lengths, held, table, free_list, free_count, q_lens, fresh, page, tokens):
    """In place: held, table, free_list, free_count. The pages last given back are the first taken."""
    n, width = table.shape
    column = torch.arange(width, device=table.device)
    anew = fresh.bool()
    begin = torch.where(anew, torch.zeros_like(lengths), lengths)
    keeps = torch.where(anew, torch.zeros_like(held), held)
    gives = torch.where(anew, held, torch.zeros_like(held)).long()
    after = begin + q_lens
    want = torch.maximum(keeps, (after + page - 1) // page)
    takes = (want - keeps).long()
    # given back: row after row, each row's pages in order, on top of the free list
    upto = torch.cumsum(gives, 0)
    mine = column[None] < gives[:, None]
    place = free_count.long() + (upto - gives)[:, None] + column[None]
    spare = free_list.shape[0]
    longer = torch.cat([free_list, free_list.new_zeros(1)])
    longer[torch.where(mine, place, torch.full_like(place, spare))] = table
    free_list.copy_(longer[:spare])
    top = free_count.long() + upto[-1]
    # taken from the top, row after row
    upto = torch.cumsum(takes, 0)
    mine = (column[None] >= keeps[:, None]) & (column[None] < want[:, None])
    place = top - 1 - ((upto - takes)[:, None] + column[None] - keeps[:, None])
    table.copy_(torch.where(mine, free_list[place.clamp(min=0)], table))
    free_count.copy_(top - upto[-1:])
    held.copy_(want)
    cu = torch.cat([q_lens.new_zeros(1), torch.cumsum(q_lens, 0).to(torch.int32)])
    token = torch.arange(tokens, device=table.device)
    req = torch.searchsorted(cu[1:].contiguous(), token, right=True)
    position = begin[req] + (token - cu[req]).to(torch.int32)
    slots = table[req, (position // page).long()] * page + position % page
    return slots, position, req.to(torch.int32), cu, after


def run(s):
    op = s["op"]
    out = {}
    if own:
        from oxr_inference_b200 import ops
    if op in ("pages", "step"):
        state = (s["lengths"], s["held"], s["table"], s["free_list"], s["free_count"], s["q_lens"], s["fresh"])
        if own:
            got = ops.step_pages(*state, page_size=s["page"], tokens=s["total"], status=s["status"])
        else:
            got = _pages(*state, s["page"], s["total"])
        slots, _, _, cu_q, ctx_lens = got
        out.update(zip(("slots", "positions", "req_of_token", "cu_q", "ctx_lens"), got))
        if op == "pages":
            return {**out, "held": s["held"], "table": s["table"], "free_list": s["free_list"], "free_count": s["free_count"]}
    else:
        slots, cu_q, ctx_lens = s["slots"], s["cu_q"], s["ctx_lens"]
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if op in ("store", "step"):
        if own:
            ops.store_kv8(s["k"], s["v"], slots, *cache, s["status"])
        else:
            _store(s["k_cache"], s["k_scale"], s["k"], slots, s["page"])
            _store(s["v_cache"], s["v_scale"], s["v"], slots, s["page"])
        out.update(k_cache=s["k_cache"], v_cache=s["v_cache"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        if op == "store":
            return out
    if own:
        out["o"] = ops.paged_attention_kv8(s["q"], *cache, cu_q=cu_q, ctx_lens=ctx_lens, block_table=s["table"], scale=s["scale"], window=s["window"],
                                           max_q_len=s["most_new"], kv_len_bound=s["longest"], status=s["status"])
    else:
        out["o"] = _attention(s["q"], *cache, cu_q, ctx_lens, s["table"], s["scale"], s["window"], s["most_new"], s["longest"])
    return out


# ------------------------------------------------------------------------------------------------------------------------------ what a pass cannot do without
def _seen_keys(case, before, new):
    """Keys that at least one of a request's new tokens sees, and (query, key) pairs, over all requests."""
    keys = pairs = 0
    w = case["window"]
    for b, q in zip(before, new):
        keys += min(b + q, q + w - 1) if w else b + q
        pairs += sum(min(b + i + 1, w) for i in range(q)) if w else q * b + q * (q + 1) // 2
    return keys, pairs


def work(case):
    before, new = _host_lengths(case)
    n, page, op = case["requests"], case["page"], case["op"]
    total = sum(new)
    size = flops = 0
    if op in ("pages", "step"):
        begin = [0 if f else b for f, b in zip(_anew(case), before)]
        # the rows' lengths, held pages and flags read, held pages, boundaries and contexts written; the pages moved; three words a token
        moved = sum(-(-b // page) for b, e in zip(before, begin) if e != b) + sum(max(0, -(-(e + q) // page) - (0 if e != b else -(-b // page))) for b, e, q in zip(before, begin, new))
        size += 4 * (4 * n + 3 * n + 2 * moved + 3 * total)
        before = begin if op == "step" else before
    if op in ("store", "step"):
        width = case["kv_heads"] * case["dim"]
        element = 2 if case["dtype"] == "bfloat16" else 4
        touched = sum(-(-(b + q) // page) - b // page for b, q in zip(before, new))
        size += 2 * total * width * (element + 1) + 2 * 2 * 4 * touched * case["kv_heads"] + 4 * total
        flops += 2 * 2 * total * width
    if op in ("attention", "step"):
        keys, pairs = _seen_keys(case, before, new)
        element = 2 if case["dtype"] == "bfloat16" else 4
        size += 2 * keys * case["kv_heads"] * case["dim"] + 2 * 4 * (keys // page + n) * case["kv_heads"] + 4 * (keys // page + n)
        size += 2 * total * case["heads"] * case["dim"] * element
        flops += 4 * pairs * case["heads"] * case["dim"]
    return {"bytes": size, "flops": flops}


# ------------------------------------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def _e4m3(x):
    """``x`` (64 bits) rounded to the nearest e4m3 number, ties to even: four significant bits, none finer than 2^-9."""
    _, exponent = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (exponent - 4).clamp(min=-9))
    return (torch.round(x / step) * step).clamp(-LARGEST, LARGEST)


def _exact_store(cache, scales, x, slots, page):
    """New codes and scales in 64 bits, page by page."""
    cache, scales, x = cache.double(), scales.double().clone(), x.double()
    by_page = {}
    for t, slot in enumerate(slots):
        by_page.setdefault(slot // page, []).append((t, slot % page))
    names = sorted(by_page)
    most = max(len(v) for v in by_page.values())
    dev = cache.device
    token = torch.tensor([[t for t, _ in by_page[p]] + [-1] * (most - len(by_page[p])) for p in names], device=dev)
    new = torch.where((token >= 0)[:, :, None, None], x[token.clamp(min=0)], torch.zeros((), dtype=torch.float64, device=dev))
    largest = new.abs().amax(dim=(1, 3))
    powers = torch.ldexp(torch.ones(1, dtype=torch.float64, device=dev), torch.arange(SMALLEST_SCALE, 121, device=dev))
    need = powers[torch.searchsorted(powers * LARGEST, largest).clamp(max=powers.numel() - 1)]   # the first that reaches it
    need = torch.where(largest > 0, need, torch.zeros_like(need))
    at = torch.tensor(names, device=dev)
    anew = torch.tensor([any(o == 0 for _, o in by_page[p]) for p in names], device=dev)
    old = scales[at]
    scale = torch.where(anew[:, None], need, torch.maximum(need, old))
    kept = cache[at]
    again = _e4m3(kept * (old / torch.where(scale > 0, scale, torch.ones_like(scale)))[:, None, :, None])
    kept = torch.where((~anew[:, None] & (scale > old))[:, None, :, None], again, kept)
    whole = cache
    whole[at] = kept
    scales[at] = scale
    slot = torch.tensor(slots, device=dev)
    mine = scales[slot // page]
    whole[slot // page, slot % page] = _e4m3(x / torch.where(mine > 0, mine, torch.ones_like(mine))[:, :, None])
    return whole, scales


def _exact_attention(q, k, v, k_scale, v_scale, tables, before, new, scale, window, page):
    """``tables``: one list of pages per request."""
    group = q.shape[1] // k.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    at = 0
    for i, (b, count) in enumerate(zip(before, new)):
        last = b + count
        ids = torch.tensor(tables[i][:-(-last // page)], device=q.device)
        keys = (k[ids].double() * k_scale[ids].double()[:, None, :, None]).flatten(0, 1)[:last]
        values = (v[ids].double() * v_scale[ids].double()[:, None, :, None]).flatten(0, 1)[:last]
        position = torch.arange(b, last, device=q.device)[:, None]
        index = torch.arange(last, device=q.device)[None]
        hidden = index > position
        if window:
            hidden = hidden | (index + window <= position)
        for h in range(q.shape[1]):
            z = q[at:at + count, h].double() @ keys[:, h // group].T * scale
            out[at:at + count, h] = torch.softmax(z.masked_fill(hidden, -math.inf), dim=-1) @ values[:, h // group]
        at += count
    return out


def exact(case, seed):
    s = prepare(case, seed)
    before, new = _host_lengths(case)
    op, page = case["op"], case["page"]
    if op == "pages":
        return None   # whole numbers
    out = {}
    if op == "step":
        # the tables in whole numbers, row by row
        tables, free = s["table"].tolist(), s["free_list"].tolist()[:int(s["free_count"])]
        anew = s["fresh"].tolist()
        tables = [row[:-(-b // page)] for row, b in zip(tables, before)]
        for i, f in enumerate(anew):
            if f:
                free += tables[i]
                tables[i] = []
        before = [0 if f else b for f, b in zip(anew, before)]
        for i, (b, q) in enumerate(zip(before, new)):
            while len(tables[i]) * page < b + q:
                tables[i].append(free.pop())
    else:
        tables = s["table"].tolist()
    slots = [tables[i][p // page] * page + p % page for i, (b, q) in enumerate(zip(before, new)) for p in range(b, b + q)]
    k, v, k_scale, v_scale = s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    if op in ("store", "step"):
        k, k_scale = _exact_store(k, k_scale, s["k"], slots, page)
        v, v_scale = _exact_store(v, v_scale, s["v"], slots, page)
        out.update(k_cache=k, v_cache=v, k_scale=k_scale, v_scale=v_scale)
    if op in ("attention", "step"):
        out["o"] = _exact_attention(s["q"], k, v, k_scale, v_scale, tables, before, new, s["scale"], s["window"], page)
    return out
