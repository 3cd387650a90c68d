"""Operators of the paged key/value cache, as cases to time and to compare: appending keys and values with their position
rotation, attention for a batch that shares a prefix, and attention over pages that a cheap score selects.

`run` computes an operator either in its plain form (elementary torch operations in 32 bits) or, where `own` is true, by the calls
that a program makes of turbovec_b200.kvcache.

What the operators compute.  A cache holds pages of `page` tokens for every key head.  Row t of a call is token j of sequence b,
where offsets[b] <= t < offsets[b + 1]; lens[b] counts the tokens of b in its own pages, those of the call among them, so the
token stands at position p = lens[b] - (offsets[b + 1] - offsets[b]) + j, in page table[b][p // page].  Rows behind the last
sequence are left as they are.

* append: q and k are rotated by the angles of position p + position_offset (tables cos and sin), k and v go into the page.  For
  every page and key head the cache keeps bounds of its keys, channel by channel: int8 (lowest, highest), outwards rounded multiples of
  a power of two, the smallest one that 127 multiples of reach the largest magnitude with (2^-24 to 2^40).
* attend: softmax attention over the shared prefix and over the sequence's own keys up to p.
* attend_selected: the query, rounded to int8 multiples of such a power of two, times whichever bound gives more, summed over the
  channels, bounds what any key of a page can score; the best over the query heads of a key head is the page's score.  The
  first and the most recent pages and the best of the others, `budget` in all, are attended to.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_E_MIN, _E_MAX = -24, 40


# ------------------------------------------------------------------------------------------------------------ the cases

def _case(name, op, dtype, heads, kv_heads, dim, page, tokens_first, seqs, new, length, **more):
    c = dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, tokens_first=tokens_first, seqs=seqs,
             new_min=new[0], new_max=new[1], len_min=length[0], len_max=length[1], shape_seed=1)
    if op == "append":
        c.update(rotary=dim, interleaved=False, position_offset=0, padding=0)
    elif op == "attend":
        c.update(prefix=0, padding=0)
    else:
        c.update(budget=32, first=1, recent=2, padding=0)
    c.update(more)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one token of one request: what a single stream pays in every layer
        _case("append_1x1", "append", "bf16", 32, 8, 128, 64, False, 1, (1, 1), (4000, 4000)),
        # one token each of a large batch, three query heads to a key head, a batch padded to a round number
        _case("append_197x1", "append", "fp16", 24, 8, 64, 16, True, 197, (1, 1), (1, 3000), padding=3),
        # pieces of prompts next to single tokens, behind a shared prefix, half of the channels rotated, pairs interleaved
        _case("append_chunks_9", "append", "bf16", 32, 8, 128, 32, True, 9, (1, 700), (700, 4000), rotary=64, interleaved=True,
              position_offset=1500),
        # whole prompts
        _case("append_prompts_4", "append", "bf16", 32, 8, 128, 64, False, 4, (7000, 9000), (9000, 9000)),
        # a handful of answers on one short document
        _case("attend_4_prefix_1000", "attend", "fp16", 8, 8, 64, 16, False, 4, (1, 1), (1, 40), prefix=1000),
        # no common prefix: requests of very different lengths
        _case("attend_48_ragged", "attend", "bf16", 32, 8, 128, 64, False, 48, (1, 1), (1, 12000)),
        # drafts of several tokens that are verified together, on a common system prompt
        _case("attend_24_drafts_prefix_8200", "attend", "bf16", 32, 8, 128, 32, True, 24, (1, 5), (5, 2000), prefix=8200, padding=2),
        # many questions on one long set of documents
        _case("attend_128_prefix_32768", "attend", "bf16", 64, 8, 128, 64, False, 128, (1, 1), (1, 1500), prefix=32768),
        # one long request
        _case("selected_1x32000", "attend_selected", "bf16", 32, 8, 128, 64, False, 1, (1, 1), (32000, 32000)),
        # drafts over requests of very different lengths, some shorter than the budget
        _case("selected_8_drafts", "attend_selected", "fp16", 12, 4, 64, 16, True, 8, (1, 4), (4, 20000), budget=48, padding=1),
        # a batch of medium lengths
        _case("selected_16_ragged", "attend_selected", "fp16", 16, 8, 128, 32, False, 16, (1, 1), (3000, 60000), budget=64, first=2, recent=4),
        # a batch of long requests
        _case("selected_48x65536", "attend_selected", "bf16", 32, 4, 128, 64, False, 48, (1, 1), (40000, 65536), budget=64),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend_selected"])
    dtype, dim, page = rng.choice(["bf16", "fp16"]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    tokens_first, padding = rng.random() < 0.5, rng.choice([0, 0, 1, 5])
    more = dict(shape_seed=rng.randrange(1 << 30), padding=padding)
    if op == "append":
        seqs = _log(rng, 1, 200)
        most = 1 if rng.random() < 0.5 else max(1, _log(rng, 1, 16000) // seqs)
        rotary = rng.choice([dim, dim, dim // 2, 32])
        more.update(rotary=rotary, interleaved=rng.random() < 0.5, position_offset=rng.choice([0, rng.randrange(5000)]))
        return _case(None, op, dtype, kv_heads * group, kv_heads, dim, page, tokens_first, seqs, (1, most), (most, most + _log(rng, 1, 4000)), **more)
    new = (1, rng.choice([1, 1, 1, 2, 4, 6]))
    if op == "attend":
        seqs = _log(rng, 1, 100)
        most = min(30000, int(2.4e8) // (seqs * new[1] * kv_heads * group))
        prefix = rng.choice([0, _log(rng, 1, most), _log(rng, min(100, most), most)])
        longest = _log(rng, 8, max(8, 80000 // seqs))
        return _case(None, op, dtype, kv_heads * group, kv_heads, dim, page, tokens_first, seqs, new, (rng.choice([1, 6]), longest),
                     prefix=prefix, **more)
    seqs = _log(rng, 1, 40)
    longest = _log(rng, 500, min(60000, 1200000 // seqs))
    budget = _log(rng, 4, max(4, min(100, int(1e8) // (seqs * new[1] * kv_heads * page * dim))))
    first = rng.randrange(0, 3)
    recent = rng.randrange(1, budget - first + 1) if rng.random() < 0.2 else min(2, budget - first)
    return _case(None, op, dtype, kv_heads * group, kv_heads, dim, page, tokens_first, seqs, new, (rng.choice([6, longest // 3]), longest),
                 budget=budget, first=first, recent=recent, **more)


def _shape(case):
    """Tokens of the call and lengths of every sequence, which belong to the case and not to the seed."""
    rng = random.Random(case["shape_seed"])
    new = [rng.randint(case["new_min"], case["new_max"]) for _ in range(case["seqs"])]
    lens = [max(_log(rng, case["len_min"], case["len_max"]), n) for n in new]
    return new, lens


def _pages_of(n, page):
    return (n + page - 1) // page


def work(case):
    new, lens = _shape(case)
    d, hq, hk, page = case["dim"], case["heads"], case["kv_heads"], case["page"]
    tokens = sum(new)
    table = 4 * sum(_pages_of(n, page) for n in lens)
    if case["op"] == "append":
        touched = sum(_pages_of(n, page) - (n - m) // page for n, m in zip(lens, new))
        old = sum(1 for n, m in zip(lens, new) if (n - m) % page)
        summary = hk * (2 * d + 4)
        nbytes = 2 * 2 * tokens * (hq + 2 * hk) * d + 4 * tokens * case["rotary"] + (touched + old) * summary + 4 * touched
        return {"bytes": nbytes, "flops": 3 * tokens * (hq + hk) * case["rotary"]}
    io = 2 * 2 * tokens * hq * d
    if case["op"] == "attend":
        pairs = sum(m * case["prefix"] + sum(n - m + j + 1 for j in range(m)) for n, m in zip(lens, new))
        keys = case["prefix"] + sum(lens)
        return {"bytes": io + 4 * tokens * hq + 2 * 2 * keys * hk * d + table + 4 * _pages_of(case["prefix"], page), "flops": 4 * d * hq * pairs}
    summaries = sum(_pages_of(n, page) for n in lens)
    scored = chosen = pages = 0
    for n, m in zip(lens, new):
        for j in range(m):
            visible = _pages_of(n - m + j + 1, page)
            scored += visible if visible > case["budget"] else 0
            chosen += (n - m + j + 1) if visible <= case["budget"] else (case["budget"] - 1) * page + (n - m + j) % page + 1
        pages += min(_pages_of(n, page), m * case["budget"]) * page
    nbytes = io + summaries * hk * (2 * d + 4) + 2 * 2 * min(pages, chosen) * hk * d + table + 4 * tokens * hk * case["budget"]
    return {"bytes": nbytes, "flops": 4 * d * hq * (chosen + scored)}


# ------------------------------------------------------------------------------------------------------------ inputs

def _exponent(amax):
    """Smallest e in [-24, 40] with amax <= 127 * 2^e."""
    m, x = torch.frexp(amax.float())
    e = x - 7 + (m > 127.0 / 128.0).to(x.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, _E_MIN)).clamp(_E_MIN, _E_MAX)


def _pow2(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)            # exact, which pow() and exp2() are not everywhere


def _bounds_of(lo, hi):
    """int8 (lowest, highest) and the power of two they are multiples of; lo and hi [..., dim]."""
    scale = _pow2(_exponent(torch.maximum(lo.abs(), hi.abs()).amax(-1).float()))
    s = scale[..., None]
    both = torch.stack([torch.floor(lo.float() / s), torch.ceil(hi.float() / s)], dim=-2)
    return both.clamp(-127, 127).to(torch.int8), scale


def prepare(case, seed):
    dev, dt = torch.device("cuda"), _DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed * 1000003 + case["shape_seed"])
    d, hq, hk, page = case["dim"], case["heads"], case["kv_heads"], case["page"]
    new, lens = _shape(case)
    tokens = sum(new) + case["padding"]
    counts = [_pages_of(n, page) for n in lens]
    width, prefix = max(counts), case.get("prefix", 0)
    prefix_pages = _pages_of(prefix, page)
    used = sum(counts) + prefix_pages
    pages = used + 3                                        # a pool has free pages too

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dt)

    # pages of a pool are handed out in any order; places of the table that a sequence does not use hold -1
    order = torch.randperm(pages, generator=gen, device=dev)[:used].to(torch.int32)
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32)
    flat = order.cpu()
    at = prefix_pages
    for b, c in enumerate(counts):
        table[b, :c] = flat[at:at + c]
        at += c
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    st = {"case": case, "table": table.to(dev), "lens": torch.tensor(lens, dtype=torch.int32, device=dev),
          "offsets": torch.tensor(offsets, dtype=torch.int32, device=dev), "prefix_pages": order[:prefix_pages]}

    # keys have channels of different size and an offset in some of them, as projections with a rotation give them
    channel = torch.exp(0.4 * torch.randn(hk, 1, d, generator=gen, device=dev)).to(dt)
    offset = (torch.randn(hk, 1, d, generator=gen, device=dev) * (torch.rand(hk, 1, d, generator=gen, device=dev) < 0.1)).to(dt)
    shape = (pages, page, hk, d) if case["tokens_first"] else (pages, hk, page, d)
    k, v = normal(*shape), normal(*shape)
    if case["tokens_first"]:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    # neighbouring tokens are alike: each page has a direction of its own
    k.mul_(channel).add_(offset).add_(normal(pages, hk, 1, d))
    st["k"], st["v"] = k, v
    if case["op"] == "append":
        k.zero_(), v.zero_()
        bounds = torch.zeros(pages, hk, 2, d, dtype=torch.int8, device=dev)
        scales = torch.full((pages, hk), 2.0 ** _E_MIN, device=dev)
        for b, (n, m) in enumerate(zip(lens, new)):        # the page that the new tokens complete holds earlier ones
            at = n - m
            if at % page:
                p = int(table[b, at // page])
                old = normal(hk, at % page, d) * channel
                k[p, :, :at % page], v[p, :, :at % page] = old, normal(hk, at % page, d)
                bounds[p], scales[p] = _bounds_of(old.amin(1), old.amax(1))
        st["q"] = normal(tokens, hq, d)
        st["k_new"], st["v_new"] = normal(tokens, hk, d).mul_(channel.view(1, hk, d)), normal(tokens, hk, d)
        st["q_out"] = torch.zeros_like(st["q"])
        far = max(lens) + case["position_offset"]
        rate = 10000.0 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64, device=dev) / case["rotary"])
        angle = torch.arange(far, dtype=torch.float64, device=dev)[:, None] * rate
        st["cos"], st["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
    else:
        if case["op"] == "attend":
            bounds, scales = None, None
        else:
            bounds, scales = _bounds_of(k.amin(2), k.amax(2))
        st["q"] = normal(tokens, hq, d)
        st["out"] = torch.zeros_like(st["q"])
        if case["op"] == "attend":
            st["lse"] = torch.zeros(tokens, hq, device=dev)
        else:
            st["pages"] = torch.full((tokens, hk, case["budget"]), -1, dtype=torch.int32, device=dev)
    st["bounds"], st["scales"] = bounds, scales
    if own:                                                 # the handles that a program keeps for its cache and its batch
        from turbovec_b200.kvcache import KVBatch, PagedKVCache
        st["cache"] = PagedKVCache(k, v, bounds, scales)
        st["batch"] = KVBatch(st["table"], st["lens"], st["offsets"])
    return st


# ------------------------------------------------------------------------------------------------------------ plain forms

def _rows(st):
    """Sequence and position of every row, and which rows belong to a sequence."""
    offsets, lens = st["offsets"].long(), st["lens"].long()
    t = torch.arange(st["q"].shape[0], device=offsets.device)
    seq = torch.searchsorted(offsets, t, right=True) - 1
    live = seq < lens.numel()
    seq = seq.clamp(max=lens.numel() - 1)
    return seq, lens[seq] - offsets[seq + 1] + t, live


def _rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    x = x.float()
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    x1, x2 = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :half], head[..., half:])
    c, s = cos[:, None], sin[:, None]
    y1, y2 = x1 * c - x2 * s, x2 * c + x1 * s
    y = torch.stack([y1, y2], -1).flatten(-2) if interleaved else torch.cat([y1, y2], -1)
    return torch.cat([y, rest], -1)


def _append(st):
    case, dt = st["case"], st["q"].dtype
    k, v, bounds, scales = st["k"], st["v"], st["bounds"], st["scales"]
    page, hk, d = case["page"], case["kv_heads"], case["dim"]
    seq, pos, live = _rows(st)
    seq, pos = seq[live], pos[live]
    cos, sin = st["cos"][pos + case["position_offset"]], st["sin"][pos + case["position_offset"]]
    st["q_out"][live] = _rotate(st["q"][live], cos, sin, case["interleaved"]).to(dt)
    kr = _rotate(st["k_new"][live], cos, sin, case["interleaved"]).to(dt)
    at, place = st["table"][seq, pos // page].long(), pos % page
    k[at, :, place] = kr
    v[at, :, place] = st["v_new"][live]
    # bounds of the new keys, page by page, widened by what the page held before
    index = at[:, None, None].expand(-1, hk, d)
    hi = torch.zeros(bounds.shape[0], hk, d, device=kr.device).scatter_reduce(0, index, kr.float(), "amax", include_self=False)
    lo = torch.zeros(bounds.shape[0], hk, d, device=kr.device).scatter_reduce(0, index, kr.float(), "amin", include_self=False)
    touched = torch.zeros(bounds.shape[0], dtype=torch.bool, device=kr.device)
    touched[at] = True
    fresh = torch.zeros_like(touched)
    fresh[at[place == 0]] = True
    scale = _pow2(_exponent(torch.maximum(lo.abs(), hi.abs()).amax(-1)))
    keep = (~fresh)[:, None]
    scale = torch.where(keep, torch.maximum(scale, scales), scale)
    s, ratio = scale[..., None], (scales / scale)[..., None]
    new_lo, new_hi = torch.floor(lo / s).clamp(-127, 127), torch.ceil(hi / s).clamp(-127, 127)
    new_lo = torch.where(keep[..., None], torch.minimum(new_lo, torch.floor(bounds[:, :, 0] * ratio)), new_lo)
    new_hi = torch.where(keep[..., None], torch.maximum(new_hi, torch.ceil(bounds[:, :, 1] * ratio)), new_hi)
    new = torch.stack([new_lo, new_hi], 2).to(torch.int8)
    bounds.copy_(torch.where(touched[:, None, None, None], new, bounds))
    scales.copy_(torch.where(touched[:, None], scale, scales))
    return _append_outputs(st)


def _append_outputs(st):
    # what is held in 8 bits goes out as the values it stands for
    return [st["q_out"], st["k"], st["v"], st["bounds"] * st["scales"][..., None, None]]


def _attend(st):
    case = st["case"]
    hq, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    g = hq // hk
    seq, pos, live = _rows(st)
    seq, pos = seq[live], pos[live]
    q = st["q"][live].float().view(-1, hk, g, d) * d ** -0.5
    tokens = q.shape[0]
    table = st["table"].long().clamp(min=0)
    k_own = st["k"][table].transpose(1, 2).flatten(2, 3).float()           # [seqs, hk, keys, d]
    v_own = st["v"][table].transpose(1, 2).flatten(2, 3).float()
    logits = torch.matmul(q, k_own[seq].transpose(-1, -2))                   # [tokens, hk, g, keys]
    hidden = torch.arange(k_own.shape[2], device=q.device) > pos[:, None]
    logits = logits.masked_fill(hidden[:, None, None], float("-inf"))
    if case["prefix"]:
        pre = st["prefix_pages"].long()
        k_pre = st["k"][pre].transpose(0, 1).flatten(1, 2)[:, :case["prefix"]].float()      # [hk, prefix, d]
        v_pre = st["v"][pre].transpose(0, 1).flatten(1, 2)[:, :case["prefix"]].float()
        shared = torch.matmul(q.transpose(0, 1).reshape(hk, tokens * g, d), k_pre.transpose(-1, -2))
        logits = torch.cat([shared.view(hk, tokens, g, -1).transpose(0, 1), logits], -1)
    top = logits.amax(-1, keepdim=True)
    w = torch.exp(logits - top)
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w[..., case["prefix"]:], v_own[seq])
    if case["prefix"]:
        shared = w[..., :case["prefix"]].transpose(0, 1).reshape(hk, tokens * g, -1)
        out = out + torch.matmul(shared, v_pre).view(hk, tokens, g, d).transpose(0, 1)
    st["out"][live] = (out / total).reshape(tokens, hq, d).to(st["out"].dtype)
    st["lse"][live] = (top + torch.log(total)).reshape(tokens, hq)
    return [st["out"], st["lse"]]


def _attend_selected(st):
    case = st["case"]
    hq, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    g, budget, first, recent = hq // hk, case["budget"], case["first"], case["recent"]
    seq, pos, live = _rows(st)
    seq, pos = seq[live], pos[live]
    q = st["q"][live].float().view(-1, hk, g, d)
    tokens = q.shape[0]
    table = st["table"].long().clamp(min=0)[seq]                             # [tokens, width]
    width = table.shape[1]
    # scores: whole numbers below 2^22 times powers of two, exact in 32 bits whatever the order
    scale = _pow2(_exponent(q.abs().amax(-1)))[..., None]                    # [tokens, hk, g, 1]
    q8 = torch.round(q / scale).clamp(-127, 127)
    lo = st["bounds"][table, :, 0].permute(0, 2, 3, 1).float()               # [tokens, hk, d, width]
    hi = st["bounds"][table, :, 1].permute(0, 2, 3, 1).float()
    score = torch.matmul(q8.clamp(min=0), hi) + torch.matmul(q8.clamp(max=0), lo)
    score = (score * scale).amax(2) * st["scales"][table].transpose(1, 2)    # [tokens, hk, width]
    # the first and the most recent pages before the others, pages that are not there behind them; equal scores go to the lower page
    at = torch.arange(width, device=q.device)
    visible = (pos + page) // page
    taken = (at < first) | (at >= (visible - recent)[:, None])
    score = score.masked_fill(taken[:, None], float("inf")).masked_fill((at >= visible[:, None])[:, None], float("-inf"))
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :budget]
    there = best < visible[:, None, None]
    chosen = torch.where(there, best, width).sort(-1).values                 # ascending, missing ones last
    if chosen.shape[-1] < budget:
        chosen = torch.cat([chosen, chosen.new_full((*chosen.shape[:2], budget - chosen.shape[-1]), width)], -1)
    there = chosen < width
    st["pages"][live] = torch.where(there, chosen, -1).to(torch.int32)
    ids = torch.gather(table[:, None].expand(-1, hk, -1), 2, chosen.clamp(max=width - 1))
    head = torch.arange(hk, device=q.device)[None, :, None]
    k, v = st["k"][ids, head].flatten(2, 3).float(), st["v"][ids, head].flatten(2, 3).float()       # [tokens, hk, budget * page, d]
    place = (chosen[..., None] * page + torch.arange(page, device=q.device)).flatten(2)
    hidden = (place > pos[:, None, None]) | ~there.repeat_interleave(page, -1)
    logits = (torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5).masked_fill(hidden[:, :, None], float("-inf"))
    w = torch.exp(logits - logits.amax(-1, keepdim=True))
    out = torch.matmul(w, v) / w.sum(-1, keepdim=True)
    st["out"][live] = out.reshape(tokens, hq, d).to(st["out"].dtype)
    return [st["out"], st["pages"]]


def run(st):
    case = st["case"]
    op = case["op"]
    if not own:
        return {"append": _append, "attend": _attend, "attend_selected": _attend_selected}[op](st)
    cache, batch = st["cache"], st["batch"]
    if op == "append":
        cache.append(batch, st["k_new"], st["v_new"], q=st["q"], q_out=st["q_out"], cos=st["cos"], sin=st["sin"],
                     interleaved=case["interleaved"], position_offset=case["position_offset"])
        return _append_outputs(st)
    if op == "attend":
        cache.attend(batch, st["q"], prefix_pages=st["prefix_pages"], prefix_len=case["prefix"], out=st["out"], lse=st["lse"])
        return [st["out"], st["lse"]]
    cache.attend_selected(batch, st["q"], budget=case["budget"], first=case["first"], recent=case["recent"], out=st["out"],
                          pages=st["pages"])
    return [st["out"], st["pages"]]


# ------------------------------------------------------------------------------------------------------------ in 64 bits

def _step(top):
    """Smallest of 2^-24 .. 2^40 that 127 multiples of reach `top` with."""
    steps = torch.tensor([2.0 ** e for e in range(_E_MIN, _E_MAX + 1)], dtype=torch.float64, device=top.device)
    return steps[torch.searchsorted(127 * steps, top.contiguous()).clamp(max=len(steps) - 1)]


def exact(case, seed):
    st = prepare(case, seed)
    d, hq, hk, page = case["dim"], case["heads"], case["kv_heads"], case["page"]
    g = hq // hk
    new, lens = _shape(case)
    table = st["table"].tolist()
    rows = [(b, lens[b] - new[b] + j) for b in range(case["seqs"]) for j in range(new[b])]
    if case["op"] == "append":
        if len(rows) > 20000:
            return None
        pos = torch.tensor([p for _, p in rows], device="cuda")
        ids = torch.tensor([table[b][p // page] for b, p in rows], device="cuda")
        half = case["rotary"] // 2
        turn = torch.complex(st["cos"].double(), st["sin"].double())[pos + case["position_offset"]][:, None]

        def turned(x):
            x = x[:len(rows)].double()
            if case["interleaved"]:
                z = torch.view_as_complex(x[..., :2 * half].unflatten(-1, (half, 2)).contiguous()) * turn
                x[..., :2 * half] = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
                x[..., :half], x[..., half:2 * half] = z.real, z.imag
            return x

        q_out, k, v = st["q_out"].double(), st["k"].double(), st["v"].double()
        q_out[:len(rows)] = turned(st["q"])
        k[ids, :, pos % page] = turned(st["k_new"])
        v[ids, :, pos % page] = st["v_new"][:len(rows)].double()
        held = k.to(st["k"].dtype).double()
        values = (st["bounds"].double() * st["scales"].double()[..., None, None])
        seen = torch.zeros(k.shape[0], dtype=torch.long, device="cuda")          # keys in each page now
        seen.scatter_reduce_(0, ids, pos % page + 1, "amax")
        for p in seen.nonzero().flatten().tolist():
            part = held[p, :, :seen[p]]
            low, high = part.amin(1), part.amax(1)
            top = torch.maximum(low.abs(), high.abs()).amax(-1)
            step = _step(top)[:, None]
            values[p, :, 0], values[p, :, 1] = torch.floor(low / step) * step, torch.ceil(high / step) * step
        return [q_out, k, v, values]

    out = st["out"].double()
    if case["op"] == "attend":
        lse = st["lse"].double()
        if work(case)["flops"] > 4e11:
            return None
        pre = st["prefix_pages"].long()
        at = 0
        for b in range(case["seqs"]):
            ids = torch.tensor(table[b][:_pages_of(lens[b], page)], device="cuda")
            pages = torch.cat([pre, ids])
            place = torch.cat([torch.arange(len(pre) * page, device="cuda") - len(pre) * page, torch.arange(len(ids) * page, device="cuda")])
            unused = (place < 0) & (place >= case["prefix"] - len(pre) * page)
            for h in range(hk):
                k, v = st["k"][pages, h].double().flatten(0, 1), st["v"][pages, h].double().flatten(0, 1)
                q = st["q"][at:at + new[b], h * g:(h + 1) * g].double()
                s = torch.einsum("tgd,nd->tgn", q, k) / math.sqrt(d)
                p = lens[b] - new[b] + torch.arange(new[b], device="cuda")
                s = s.masked_fill((unused | (place > p[:, None]))[:, None], float("-inf"))
                out[at:at + new[b], h * g:(h + 1) * g] = torch.softmax(s, -1) @ v
                lse[at:at + new[b], h * g:(h + 1) * g] = torch.logsumexp(s, -1)
            at += new[b]
        return [out, lse]

    if len(rows) * hk > 2000:
        return None
    pages = st["pages"]
    for t, (b, p) in enumerate(rows):
        n = p // page + 1
        ids = torch.tensor(table[b][:n], device="cuda")
        low, high = st["bounds"][ids].double().unbind(2)                          # [n, hk, d]
        for h in range(hk):
            q = st["q"][t, h * g:(h + 1) * g].double()
            step = _step(q.abs().amax(-1))[:, None]
            q8 = torch.round(q / step)
            bound = (torch.maximum(q8 * low[:, None, h], q8 * high[:, None, h]).sum(-1) * step[:, 0]).amax(1) * st["scales"][ids, h].double()
            if n <= case["budget"]:
                chosen = list(range(n))
            else:
                middle = range(case["first"], n - case["recent"])
                value = bound.tolist()
                best = sorted(middle, key=lambda i: (-value[i], i))[:case["budget"] - case["first"] - case["recent"]]
                chosen = sorted([*range(case["first"]), *best, *range(n - case["recent"], n)])
            pages[t, h] = -1
            pages[t, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
            pick = torch.tensor(chosen, device="cuda")
            k, v = st["k"][ids[pick], h].double().flatten(0, 1), st["v"][ids[pick], h].double().flatten(0, 1)
            s = q @ k.T / math.sqrt(d)
            s = s.masked_fill((pick[:, None] * page + torch.arange(page, device="cuda")).flatten() > p, float("-inf"))
            out[t, h * g:(h + 1) * g] = torch.softmax(s, -1) @ v
    return [out, pages]
