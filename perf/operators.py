"""The paged 8-bit KV cache's operators, whose speed is measured: what a program that serves many requests at once does
with its cache in a step, from the requests' lengths to the attention over the pages.

A cache's page holds `page` tokens: K codes int8 [pages, kv_heads, page, head_dim], V codes int8 [pages, kv_heads,
head_dim, page], one F32 scale for each page and KV head (k_scale, v_scale [pages, kv_heads]; a value is its code times
that scale) and, for the selection, the smallest and the largest K code of every dimension (low, high [pages, kv_heads,
head_dim]). A request's row of the table names its pages in order. A case's "path" says which operators a pass makes:

  plan     the requests' lengths before and after a step: pages taken from and given back to the ring of free ones, the
           table's new entries, a slot, position and request for every new token, and the list of the pages they touch
  store    the new tokens' K and V rows quantized into the pages they touch, then those pages read back as values
  attend   attention over each request's pages, one token or many a request, causal
  sparse   for every query and KV head the pages with the largest bound on a logit, then attention over those alone
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # The smallest call: a decode step of 64 requests, each with one new token, every 64th of them on a new page.
        {"name": "plan_64_requests", "path": "plan", "requests": 64, "page": 64, "longest": 8192, "fresh": 1},
        # A step of a full server: requests that end, that begin with prompts and that go on, 16-token pages.
        {"name": "plan_1000_requests", "path": "plan", "requests": 1000, "page": 16, "longest": 8192, "fresh": 300},
        # A decode step's rows of 64 requests into the cache, each at its own place in its last page.
        {"name": "store_64_tokens", "path": "store", "requests": 64, "page": 64, "longest": 4096, "fresh": 1, "kv_heads": 8, "head_dim": 128,
         "dtype": "bf16"},
        # Prompt chunks of odd lengths from seven requests, most of them beginning inside a page.
        {"name": "store_prompts", "path": "store", "requests": 7, "page": 32, "longest": 4096, "fresh": 2048, "kv_heads": 8, "head_dim": 256,
         "dtype": "f16"},
        # One user's decode step over 8192 tokens, F32 activations (16 heads over 8 KV heads of 256).
        {"name": "attend_1_request_8192", "path": "attend", "requests": 1, "page": 64, "longest": 8192, "fresh": 1, "heads": 16, "kv_heads": 8,
         "head_dim": 256, "dtype": "f32", "window": 0, "softcap": 0.0, "sinks": False},
        # The ordinary decode step of a server: 32 requests of ragged lengths up to 16384 tokens.
        {"name": "attend_32_requests", "path": "attend", "requests": 32, "page": 64, "longest": 16384, "fresh": 1, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "dtype": "bf16", "window": 0, "softcap": 0.0, "sinks": False},
        # One request with a very long context.
        {"name": "attend_1_request_131072", "path": "attend", "requests": 1, "page": 128, "longest": 131072, "fresh": 1, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "window": 0, "softcap": 0.0, "sinks": False},
        # Drafted tokens being verified: up to five a request, small pages, a window, and heads with sinks (14 heads over 2).
        {"name": "attend_drafts_window_sinks", "path": "attend", "requests": 9, "page": 16, "longest": 2777, "fresh": 5, "heads": 14,
         "kv_heads": 2, "head_dim": 64, "dtype": "f16", "window": 1024, "softcap": 0.0, "sinks": True},
        # A prompt's second chunk of 2048 tokens: the largest products.
        {"name": "attend_prompt_2048", "path": "attend", "requests": 1, "page": 64, "longest": 4096, "fresh": 2048, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "dtype": "bf16", "window": 0, "softcap": 0.0, "sinks": False},
        # Prompts and decode steps of ragged lengths in one call, with a softcap (16 heads over 8 KV heads of 256).
        {"name": "attend_ragged_softcap", "path": "attend", "requests": 6, "page": 32, "longest": 2500, "fresh": 777, "heads": 16, "kv_heads": 8,
         "head_dim": 256, "dtype": "bf16", "window": 0, "softcap": 50.0, "sinks": False},
        # Decode steps over long contexts that read 64 of up to 1024 pages.
        {"name": "sparse_8_requests_65536", "path": "sparse", "requests": 8, "page": 64, "longest": 65536, "fresh": 1, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "dtype": "bf16", "keep": 64},
        # A short follow-up prompt over a long context, each of its tokens with pages of its own choice.
        {"name": "sparse_100_tokens", "path": "sparse", "requests": 2, "page": 32, "longest": 20000, "fresh": 100, "heads": 16, "kv_heads": 4,
         "head_dim": 128, "dtype": "f16", "keep": 48},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    path = rng.choice(["plan", "store", "attend", "attend", "attend", "sparse"])
    page = rng.choice([16, 32, 64, 128])
    if path == "plan":
        return {"path": path, "requests": _log(rng, 1, 1000), "page": page, "longest": _log(rng, 64, 8192), "fresh": rng.choice([1, _log(rng, 2, 300)])}
    if path == "store":
        fresh = rng.choice([1, _log(rng, 2, 2048)])
        return {"path": path, "requests": _log(rng, 1, 64 if fresh == 1 else 7), "page": page, "longest": max(fresh, _log(rng, 16, 4096)), "fresh": fresh,
                "kv_heads": rng.choice([1, 2, 4, 8]), "head_dim": rng.choice([64, 128, 256]), "dtype": rng.choice(list(DTYPES))}
    heads, kv_heads, head_dim = rng.choice([(16, 8, 256), (8, 4, 256), (32, 8, 128), (16, 4, 128), (28, 4, 128), (12, 1, 128), (14, 2, 64), (16, 16, 64)])
    dtype = rng.choice(list(DTYPES))
    if path == "attend":
        base = {"heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "window": rng.choice([0, 0, _log(rng, 16, 4096)]),
                "softcap": rng.choice([0.0, 0.0, 30.0]), "sinks": rng.random() < 0.25}
        if rng.random() < 0.6:
            requests = _log(rng, 1, 64)
            return {"path": path, "requests": requests, "page": page, "longest": _log(rng, 8, min(131072, 300000 // requests)), "fresh": rng.choice([1, 1, _log(rng, 2, 8)]),
                    **base}
        requests = _log(rng, 1, 6)
        fresh = _log(rng, 9, 2000 // requests)
        return {"path": path, "requests": requests, "page": page, "longest": max(fresh, _log(rng, 16, 4000)), "fresh": fresh, **base}
    requests = _log(rng, 1, 8)
    return {"path": path, "requests": requests, "page": page, "longest": _log(rng, 512, 65536 // requests), "fresh": rng.choice([1, 1, _log(rng, 2, 32 // requests + 2)]),
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "keep": _log(rng, 4, 64)}


# ---------------------------------------------------------------- inputs


def _requests(case):
    """(before, after) of every request: the first is the longest and has the most new tokens, the others' are spread over
    their ranges' logarithms. With five or more the last one has nothing new, and a plan's every sixth has ended."""
    rng = random.Random(case["requests"] * 1000003 + case["longest"] * 1009 + case["fresh"])
    before, after = [], []
    for r in range(case["requests"]):
        length = case["longest"] if r == 0 else _log(rng, max(1, case["longest"] // 8), case["longest"])
        new = case["fresh"] if r == 0 or case["fresh"] == 1 else _log(rng, 1, case["fresh"])
        new = min(new, length)
        if r == case["requests"] - 1 and case["requests"] >= 5:
            new = 0
        if case["path"] == "plan" and r % 6 == 5:
            before.append(length), after.append(0)
        else:
            before.append(length - new), after.append(length)
    return before, after


def _ceil(a, b):
    return -(-a // b)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(before, after):
    starts = [0]
    for b, a in zip(before, after):
        starts.append(starts[-1] + max(a - b, 0))
    return starts


def _cache(case, pages, g):
    """Codes as quantized normal values have them; a page's keys share a direction, as neighbouring tokens' do."""
    heads, d, page = case["kv_heads"], case["head_dim"], case["page"]
    cache = {}
    for name, shape, axes in (("k", (pages, heads, page, d), (2, 3)), ("v", (pages, heads, d, page), (2, 3))):
        codes = torch.empty(shape, dtype=torch.int8, device="cuda")
        scales = torch.empty((pages, heads), dtype=torch.float32, device="cuda")
        step = max(1, (1 << 27) // (heads * d * page))
        for at in range(0, pages, step):
            x = torch.randn((min(step, pages - at),) + shape[1:], device="cuda", generator=g)
            if name == "k":
                x += 0.7 * torch.randn((x.shape[0], heads, 1, d), device="cuda", generator=g)
            s = x.abs().amax(axes) / 127.0
            codes[at:at + step] = torch.round(x / s[:, :, None, None]).to(torch.int8)
            scales[at:at + step] = s
        cache[name], cache[name + "_scale"] = codes, scales
    cache["low"], cache["high"] = cache["k"].amin(2), cache["k"].amax(2)
    return cache


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    before, after = _requests(case)
    page, requests = case["page"], case["requests"]
    starts = _starts(before, after)
    tokens = starts[-1]
    s["tokens"], s["most"] = tokens, max(1, max(a - b for b, a in zip(before, after)))
    s["before"], s["after"], s["starts"] = _ints(before), _ints(after), _ints(starts)
    width = _ceil(case["longest"], page) + 1
    held = [_ceil(b if case["path"] == "plan" else a, page) for b, a in zip(before, after)]
    used = sum(held)
    pages = used + max(1, sum(max(0, _ceil(a, page) - _ceil(b, page)) for b, a in zip(before, after)))
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    # The first `used` pages of a random order are the requests', the others are free.
    counts = torch.tensor(held, device="cuda")
    ends = torch.cumsum(counts, 0)
    column = torch.arange(width, device="cuda")
    place = (ends - counts)[:, None] + column
    table = torch.where(column < counts[:, None], order[place.clamp(max=pages - 1)], torch.full_like(order[:1], -1))
    s["table"] = table.contiguous()
    if case["path"] == "plan":
        head = int(seed) % pages  # where the ring's first free page lies
        ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        free = pages - used
        ring[(head + torch.arange(free, device="cuda")) % pages] = order[used:]
        s["ring"], s["counters"] = ring, _ints([head, free, 0])
        return s
    s["cache"] = _cache(case, pages, g)
    s["lengths"] = s["after"]
    dtype, d = DTYPES[case["dtype"]], case["head_dim"]
    if case["path"] == "store":
        work = [(r, j, starts[r] + max(j * page - b, 0), max(b - j * page, 0), min(a, (j + 1) * page) - max(b, j * page))
                for r, (b, a) in enumerate(zip(before, after)) if a > b for j in range(b // page, (a - 1) // page + 1)]
        work = _ints(work)
        s["work"] = torch.stack([table[work[:, 0].long(), work[:, 1].long()], work[:, 2], work[:, 3], work[:, 4]], 1).contiguous()
        # Most of a step's rows lie within the range that their page already has.
        for name in ("k", "v"):
            s[name] = (torch.randn((tokens, case["kv_heads"], d), device="cuda", generator=g) * 0.9).to(dtype)
        return s
    s["q"] = (torch.randn((tokens, case["heads"], d), device="cuda", generator=g) * 1.5).to(dtype)
    s["scale"] = 1.0 / math.sqrt(d)
    s["sinks"] = torch.randn(case["heads"], device="cuda", generator=g) if case.get("sinks") else None
    return s


# ---------------------------------------------------------------- the passes


def run(s):
    if own:
        return _own(s)
    return {"plan": _plan, "store": _store, "attend": _attend, "sparse": _sparse}[s["path"]](s)


def _own(s):
    from llmp_amd import ops
    if s["path"] == "plan":
        plan = ops.paged_plan(s["before"], s["after"], s["table"], s["ring"], s["counters"], s["page"], s["tokens"])
        return {"table": s["table"], "ring": s["ring"], **{k: plan[k] for k in ("starts", "lengths", "slots", "positions", "requests", "work", "counters")}}
    cache = s["cache"]
    if s["path"] == "store":
        ops.paged_store(cache, s["k"], s["v"], s["work"])
        pages = s["work"][:, 0]
        k, v = ops.paged_read(cache, pages, s["k"].dtype)
        return {"k": k, "v": v, "k_scale": cache["k_scale"], "v_scale": cache["v_scale"], "low": cache["low"], "high": cache["high"]}
    if s["path"] == "attend":
        return {"out": ops.paged_attend(cache, s["q"], s["table"], s["lengths"], s["starts"], s["scale"], window=s["window"], softcap=s["softcap"],
                                        sinks=s["sinks"], most=s["most"])}
    lists = ops.paged_select(cache, s["q"], s["table"], s["lengths"], s["starts"], s["keep"], most=s["most"])
    out = ops.paged_attend(cache, s["q"], s["table"], s["lengths"], s["starts"], s["scale"], lists=lists, most=s["most"])
    return {"lists": lists, "out": out}


def _plan(s):
    page, tokens, ring = s["page"], s["tokens"], s["ring"]
    before, after = s["before"].clamp(min=0), s["after"].clamp(min=0)
    head, free = s["counters"][0], s["counters"][1]
    width = s["table"].shape[1]
    fresh = (after - before).clamp(min=0)
    zero = torch.zeros_like(before[:1])
    starts = torch.cat([zero, torch.cumsum(fresh, 0).to(torch.int32)])
    first = torch.div(before + page - 1, page, rounding_mode="floor").clamp(max=width)
    last = torch.div(after + page - 1, page, rounding_mode="floor").clamp(max=width)
    need, give = (last - first).clamp(min=0), (first - last).clamp(min=0)
    need_end = torch.cumsum(need, 0).to(torch.int32)
    give_end = torch.cumsum(give, 0).to(torch.int32)
    got = torch.minimum(need, (free - (need_end - need)).clamp(min=0))
    lengths = torch.where(after <= before, after, torch.minimum(after, torch.maximum(before, (first + got) * page)))
    taken = torch.minimum(need_end[-1], free)
    column = torch.arange(width, dtype=torch.int32, device=before.device)
    new = (column >= first[:, None]) & (column < (first + got)[:, None])
    at = (head + (need_end - need)[:, None] + column - first[:, None]) % ring.numel()
    table = torch.where(new, ring[at.clamp(min=0).long()], s["table"])
    gone = (column >= last[:, None]) & (column < first[:, None])
    at = (head + free + (give_end - give)[:, None] + column - last[:, None]) % ring.numel()
    into = torch.where(gone, at, torch.full_like(at, ring.numel())).long()
    ring = torch.cat([ring, zero]).scatter(0, into.reshape(-1), s["table"].reshape(-1))[:-1]
    t = torch.arange(tokens, dtype=torch.int32, device=before.device)
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=before.numel() - 1)
    real = t < starts[-1]
    positions = torch.where(real, before[r] + t - starts[r], torch.full_like(t, -1))
    j = torch.div(positions, page, rounding_mode="floor").clamp(0, width - 1)
    slots = torch.where(real & (positions < lengths[r]), table[r, j.long()] * page + positions % page, torch.full_like(t, -1))
    requests = torch.where(real, r.to(torch.int32), torch.full_like(t, -1))
    # The pages touched, in order: a column of the table is one where it holds new tokens.
    touched = (column >= torch.div(before, page, rounding_mode="floor")[:, None]) & (column * page < lengths[:, None]) & (lengths > before)[:, None]
    count = min(tokens, 2 * before.numel() + tokens // page)
    index = torch.cumsum(touched.reshape(-1), 0) - 1
    low = torch.maximum(column * page, before[:, None])
    item = torch.stack([table, starts[:-1, None] + low - before[:, None], low - column * page, torch.minimum(lengths[:, None], (column + 1) * page) - low], 2)
    index = torch.where(touched.reshape(-1), index, torch.full_like(index, count))
    work = torch.zeros((count + 1, 4), dtype=torch.int32, device=before.device)
    work[:, 0] = -1
    work = work.scatter(0, index[:, None].expand(-1, 4), item.reshape(-1, 4))[:-1]
    missing = (after - lengths).clamp(min=0).sum().to(torch.int32)
    counters = torch.stack([(head + taken) % ring.numel(), free - taken + give_end[-1], missing])
    return {"table": table, "ring": ring, "starts": starts, "lengths": lengths, "slots": slots, "positions": positions, "requests": requests,
            "work": work, "counters": counters}


def _store(s):
    cache, work, page = s["cache"], s["work"], s["page"]
    at, row, held, count = (work[:, i] for i in range(4))
    at = at.long()
    slot = torch.arange(page, device=work.device)
    new = (slot >= held[:, None]) & (slot < (held + count)[:, None])
    old = slot < held[:, None]
    rows = (row[:, None] + slot - held[:, None]).clamp(0, s["tokens"] - 1).long()
    for name in ("k", "v"):
        x = s[name].float()[rows]  # [items, page, heads, d]
        size = torch.where(torch.isfinite(x) & new[:, :, None, None], x.abs(), torch.zeros_like(x)).amax((1, 3))
        before = torch.where(held[:, None] > 0, cache[name + "_scale"][at], torch.zeros_like(size))
        scale = torch.maximum(before, size / 127.0)
        factor = torch.where(scale > before, before / scale, torch.ones_like(scale))
        fresh = torch.where(scale[:, None, :, None] > 0, x / scale[:, None, :, None], torch.zeros_like(x))
        fresh = torch.nan_to_num(torch.round(fresh).clamp(-127, 127), nan=0.0)
        codes = cache[name][at].float()
        codes = codes if name == "k" else codes.transpose(2, 3)
        codes = torch.where(old[:, None, :, None], torch.round(codes * factor[:, :, None, None]), codes)
        codes = torch.where(new[:, None, :, None], fresh.transpose(1, 2), codes)
        if name == "k":
            none = ~new[:, :, None, None]
            for part, far, pick, best in (("low", 1e9, torch.amin, torch.minimum), ("high", -1e9, torch.amax, torch.maximum)):
                edge = pick(fresh.masked_fill(none, far), 1)
                had = torch.round(cache[part][at].float() * factor[:, :, None])
                cache[part][at] = torch.where(held[:, None, None] > 0, best(edge, had), edge).to(torch.int8)
        cache[name][at] = (codes if name == "k" else codes.transpose(2, 3)).to(torch.int8)
        cache[name + "_scale"][at] = scale
    k = cache["k"][at].float() * cache["k_scale"][at][:, :, None, None]
    v = cache["v"][at].float().transpose(2, 3) * cache["v_scale"][at][:, :, None, None]
    dtype = s["k"].dtype
    return {"k": k.to(dtype), "v": v.to(dtype).contiguous(), "k_scale": cache["k_scale"], "v_scale": cache["v_scale"], "low": cache["low"],
            "high": cache["high"]}


def _padded(s):
    """The queries a request at a time: [requests, kv_heads, most * group, d] in 32 bits, the positions [requests, most]
    (-1 where a request has fewer tokens), and every token's request and place."""
    q, starts, lengths = s["q"].float(), s["starts"], s["lengths"]
    tokens, heads, d = q.shape
    kv_heads, most = s["cache"]["k"].shape[1], s["most"]
    place = torch.arange(most, device=q.device)
    fresh = starts[1:] - starts[:-1]
    rows = (starts[:-1, None] + place).clamp(max=tokens - 1).long()
    x = q[rows].view(-1, most, kv_heads, heads // kv_heads, d).transpose(1, 2).reshape(-1, kv_heads, most * (heads // kv_heads), d)
    position = torch.where(place < fresh[:, None], (lengths - fresh)[:, None] + place, torch.full_like(rows, -1))
    t = torch.arange(tokens, device=q.device)
    request = torch.searchsorted(starts[1:].contiguous(), t.to(torch.int32), right=True).clamp(max=fresh.numel() - 1)
    return x, position, request, t - starts[request]


def _softmax(s, score, sees, sinks):
    """exp(score - max) of what is seen, and one over its sum (zero where nothing is)."""
    if s.get("softcap"):
        score = s["softcap"] * torch.tanh(score / s["softcap"])
    score = score.masked_fill(~sees, -math.inf)
    top = score.amax(-1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks - top)
    return p, torch.where(total > 0, 1.0 / total, torch.zeros_like(total))


def _attend(s):
    cache, page = s["cache"], s["page"]
    kv_heads, d = cache["k"].shape[1], cache["k"].shape[3]
    group = s["heads"] // kv_heads
    x, position, request, place = _padded(s)
    requests, most = position.shape
    at = s["table"].clamp(min=0).long()
    k = (cache["k"][at].float() * cache["k_scale"][at][..., None, None]).transpose(1, 2).reshape(requests, kv_heads, -1, d)
    score = torch.matmul(x, k.transpose(2, 3).contiguous()) * s["scale"]
    del k
    j = torch.arange(score.shape[3], device=x.device)
    sees = j <= position[:, :, None]
    if s["window"]:
        sees &= j > position[:, :, None] - s["window"]
    sees = sees[:, None, :, None, :].expand(-1, -1, -1, group, -1).reshape(requests, 1, most * group, -1)
    sinks = s["sinks"]
    if sinks is not None:
        sinks = sinks.view(1, kv_heads, 1, group).expand(-1, -1, most, -1).reshape(1, kv_heads, most * group, 1)
    p, scale = _softmax(s, score, sees, sinks)
    del score
    v = (cache["v"][at].float() * cache["v_scale"][at][..., None, None]).permute(0, 2, 1, 4, 3).reshape(requests, kv_heads, -1, d)
    out = torch.matmul(p, v) * scale
    out = out.view(requests, kv_heads, most, group, d).transpose(1, 2).reshape(requests, most, s["heads"], d)
    return {"out": out[request, place].to(s["q"].dtype)}


def _select(s):
    cache, page, keep = s["cache"], s["page"], s["keep"]
    kv_heads, d = cache["k"].shape[1], cache["k"].shape[3]
    x, position, request, place = _padded(s)
    requests, most = position.shape
    size = x.abs().amax(-1, keepdim=True)
    unit = size / 127.0
    codes = torch.where(unit > 0, torch.round(x / unit).clamp(-127, 127), torch.zeros_like(x))
    at = s["table"].clamp(min=0).long()
    high = cache["high"][at].float().permute(0, 2, 3, 1).contiguous()  # [requests, kv_heads, d, pages]
    low = cache["low"][at].float().permute(0, 2, 3, 1).contiguous()
    whole = torch.matmul(codes.clamp(min=0), high) + torch.matmul(codes.clamp(max=0), low)  # whole numbers below 2^24
    score = (whole * unit) * cache["k_scale"][at].transpose(1, 2)[:, :, None, :]
    score = score.view(requests, kv_heads, most, -1, score.shape[3]).amax(3)  # the largest of the group's heads
    score = torch.nan_to_num(score, nan=-math.inf, posinf=3e38)
    score, n = score.transpose(1, 2)[request, place], torch.div(position[request, place], page, rounding_mode="floor") + 1
    j = torch.arange(score.shape[2], device=x.device)
    score = torch.where((j < 1) | (j == n[:, None, None] - 1), math.inf, score).masked_fill(j >= n[:, None, None], -math.inf)
    best = torch.sort(score, dim=2, descending=True, stable=True)[1][:, :, :keep]
    best = torch.where(torch.arange(best.shape[2], device=x.device) < n[:, None, None], best, torch.full_like(best, 1 << 30))
    best = torch.sort(best, dim=2)[0]
    lists = torch.full((score.shape[0], kv_heads, keep), -1, dtype=torch.int32, device=x.device)
    lists[:, :, :best.shape[2]] = torch.where(best < 1 << 30, best, torch.full_like(best, -1)).to(torch.int32)
    return lists, position[request, place], request


def _sparse(s):
    cache, page = s["cache"], s["page"]
    lists, position, request = _select(s)
    tokens, kv_heads, keep = lists.shape
    d = cache["k"].shape[3]
    at = s["table"][request[:, None, None], lists.clamp(min=0).long()].clamp(min=0).long()
    head = torch.arange(kv_heads, device=at.device)[None, :, None]
    k = (cache["k"][at, head].float() * cache["k_scale"][at, head][..., None, None]).view(tokens, kv_heads, keep * page, d)
    x = s["q"].float().view(tokens, kv_heads, -1, d)
    score = torch.matmul(x, k.transpose(2, 3).contiguous()) * s["scale"]
    j = lists[..., None] * page + torch.arange(page, device=at.device)
    sees = (lists[..., None] >= 0) & (j <= position[:, None, None, None])
    p, scale = _softmax(s, score, sees.view(tokens, kv_heads, 1, keep * page), None)
    v = (cache["v"][at, head].float() * cache["v_scale"][at, head][..., None, None]).transpose(3, 4).reshape(tokens, kv_heads, keep * page, d)
    return {"lists": lists, "out": (torch.matmul(p, v) * scale).view(tokens, -1, d).to(s["q"].dtype)}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    before, after = _requests(case)
    page = case["page"]
    fresh = [max(0, a - b) for b, a in zip(before, after)]
    tokens = sum(fresh)
    touched = sum((a - 1) // page - b // page + 1 for b, a in zip(before, after) if a > b)
    if case["path"] == "plan":
        moved = sum(abs(_ceil(a, page) - _ceil(b, page)) for b, a in zip(before, after))
        # Lengths in and out, starts; slots, positions and requests; the touched pages' items; a table entry and a ring entry a page that moves.
        return {"bytes": 16 * case["requests"] + 12 * tokens + 16 * touched + 8 * moved, "flops": 0}
    d, kv_heads, size = case["head_dim"], case["kv_heads"], SIZES[case["dtype"]]
    if case["path"] == "store":
        # The rows in and their codes out, the edges of K's codes and the scales in and out; the touched pages' codes in and values out.
        row = kv_heads * d
        return {"bytes": 2 * tokens * row * (size + 1) + touched * (4 * row + 16 * kv_heads) + 2 * touched * page * row * (1 + size),
                "flops": 4 * tokens * row}
    heads = case["heads"]
    ends = 2 * tokens * heads * d * size  # the queries in, the values out
    if case["path"] == "attend":
        window = case["window"] or 1 << 30
        seen = sum(min(a, window + n - 1) for a, n in zip(after, fresh) if n)
        pairs = sum(min(p + 1, window) for b, a in zip(before, after) for p in range(b, a))
        return {"bytes": 2 * seen * kv_heads * d + ends + seen // page * (4 + 8 * kv_heads), "flops": 4 * pairs * heads * d}
    pages = sum(_ceil(a, page) for a, n in zip(after, fresh) if n)
    picked = sum(min(case["keep"], p // page + 1) for b, a in zip(before, after) for p in range(b, a))  # of every KV head
    read = min(picked, sum(min(_ceil(a, page), n * case["keep"]) for a, n in zip(after, fresh)))
    scored = sum(p // page + 1 for b, a in zip(before, after) for p in range(b, a))
    return {"bytes": pages * kv_heads * (2 * d + 4) + 2 * read * page * kv_heads * d + ends + 4 * tokens * kv_heads * case["keep"],
            "flops": 4 * scored * heads * d + 4 * picked * page * heads * d}


# ---------------------------------------------------------------- the definitions, in 64 bits


def _exact_plan(s):
    page, ring, table = s["page"], s["ring"].tolist(), s["table"].tolist()
    head, free, _ = s["counters"].tolist()
    size, left, put = len(ring), free, 0
    taken = list(ring)
    starts, lengths, slots, positions, requests, items = [0], [], [], [], [], []
    for r, (b, a) in enumerate(zip(s["before"].tolist(), s["after"].tolist())):
        have, want = _ceil(b, page), _ceil(a, page)
        for j in range(want, have):
            ring[(head + free + put) % size] = table[r][j]
            put += 1
        n = have
        while n < want and left:
            table[r][n] = taken[(head + free - left) % size]
            left, n = left - 1, n + 1
        length = a if a <= b else min(a, max(b, n * page))
        lengths.append(length)
        for p in range(b, a):
            slots.append(table[r][p // page] * page + p % page if p < length else -1)
            positions.append(p), requests.append(r)
        for j in range(b // page, _ceil(length, page) if length > b else 0):
            items.append([table[r][j], starts[-1] + max(j * page - b, 0), max(b - j * page, 0), min(length, j * page + page) - max(b, j * page)])
        starts.append(starts[-1] + max(a - b, 0))
    count = min(s["tokens"], 2 * s["requests"] + s["tokens"] // page)
    items += [[-1, 0, 0, 0]] * (count - len(items))
    missing = sum(max(a - n, 0) for a, n in zip(s["after"].tolist(), lengths))
    out = {"table": table, "ring": ring, "starts": starts, "lengths": lengths, "slots": slots, "positions": positions, "requests": requests,
           "work": items, "counters": [(head + free - left) % size, left + put, missing]}
    return {k: torch.tensor(v, dtype=torch.int32) for k, v in out.items()}


def _exact_store(s):
    cache, page = s["cache"], s["page"]
    k_out, v_out = [], []
    for at, row, held, count in s["work"].tolist():
        for name, out in (("k", k_out), ("v", v_out)):
            x = s[name][row:row + count].double().transpose(0, 1)  # [heads, count, d]
            old = cache[name + "_scale"][at].double() if held else torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
            # A scale is held in 32 bits.
            scale = torch.maximum(old, (x.abs().amax((1, 2)) / 127.0).float().double())
            codes = cache[name][at].double()
            codes = codes if name == "k" else codes.transpose(1, 2).contiguous()
            factor = (old / scale)[:, None, None]
            codes[:, :held] = torch.round(codes[:, :held] * factor)
            codes[:, held:held + count] = torch.round(x / scale[:, None, None]).clamp(-127, 127)
            if name == "k":
                new = codes[:, held:held + count]
                low, high = new.amin(1), new.amax(1)
                if held:
                    low = torch.minimum(low, torch.round(cache["low"][at].double() * factor[:, :, 0]))
                    high = torch.maximum(high, torch.round(cache["high"][at].double() * factor[:, :, 0]))
                cache["low"][at], cache["high"][at] = low.to(torch.int8), high.to(torch.int8)
            cache[name + "_scale"][at] = scale.float()
            out.append(codes * scale[:, None, None])
    return {"k": torch.stack(k_out), "v": torch.stack(v_out), "k_scale": cache["k_scale"].double(), "v_scale": cache["v_scale"].double(),
            "low": cache["low"], "high": cache["high"]}


def _exact_row(s, r, head, j, t0, t1):
    """Attention of tokens t0 to t1 of request r in the heads of KV head `head` over the keys at positions j."""
    cache, page = s["cache"], s["page"]
    at = s["table"][r].long()[j // page]
    k = cache["k"][at, head, j % page].double() * cache["k_scale"][at, head].double()[:, None]
    v = cache["v"][at, head, :, j % page].double() * cache["v_scale"][at, head].double()[:, None]
    start, end, length = s["starts"][r].item(), s["starts"][r + 1].item(), s["lengths"][r].item()
    group = s["heads"] // cache["k"].shape[1]
    q = s["q"][start + t0:start + t1, head * group:(head + 1) * group].double()
    position = length - (end - start) + torch.arange(t0, t1, device=q.device)
    score = torch.matmul(q, k.T) * s["scale"]
    if s.get("softcap"):
        score = s["softcap"] * torch.tanh(score / s["softcap"])
    hidden = j > position[:, None]
    if s.get("window"):
        hidden = hidden | (j <= position[:, None] - s["window"])
    score = score.masked_fill(hidden[:, None, :], -math.inf)
    if s.get("sinks") is not None:
        score = torch.cat([score, s["sinks"][head * group:(head + 1) * group].double()[None, :, None].expand(t1 - t0, -1, 1)], 2)
        v = torch.cat([v, torch.zeros_like(v[:1])])
    return torch.nan_to_num(torch.matmul(torch.softmax(score, 2), v))


def exact(case, seed):
    s = prepare(case, seed)
    if case["path"] == "plan":
        return _exact_plan(s)
    if case["path"] == "store":
        return _exact_store(s)
    device = s["q"].device
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=device)
    group = s["heads"] // s["kv_heads"]
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    lists = None
    if case["path"] == "sparse":
        if s["tokens"] * s["kv_heads"] > 2000:
            return None
        lists = _exact_lists(s)
    for r, length in enumerate(lengths):
        n = starts[r + 1] - starts[r]
        for head in range(s["kv_heads"]):
            step = n if n == 0 else (1 if lists is not None else max(1, (1 << 27) // (length * group)))
            for t0 in range(0, n, step or 1):
                t1 = min(n, t0 + step)
                if lists is None:
                    j = torch.arange(length, device=device)
                else:
                    picked = lists[starts[r] + t0, head]
                    picked = picked[picked >= 0].long()
                    j = (picked[:, None] * s["page"] + torch.arange(s["page"], device=device)).reshape(-1)
                    j = j[j < length]
                out[starts[r] + t0:starts[r] + t1, head * group:(head + 1) * group] = _exact_row(s, r, head, j, t0, t1)
    return {"out": out} if lists is None else {"lists": lists, "out": out}


def _exact_lists(s):
    """The pages by their definition: a page's score is whole numbers' sum times the two scales, each product rounded to
    the 32 bits that it is held in."""
    cache, page, keep = s["cache"], s["page"], s["keep"]
    kv_heads = cache["k"].shape[1]
    group = s["heads"] // kv_heads
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    lists = torch.full((s["tokens"], kv_heads, keep), -1, dtype=torch.int32, device=s["q"].device)
    for r, length in enumerate(lengths):
        for t in range(starts[r], starts[r + 1]):
            n = (length - (starts[r + 1] - t)) // page + 1
            at = s["table"][r, :n].long()
            for head in range(kv_heads):
                q = s["q"][t, head * group:(head + 1) * group].double()
                unit = (q.abs().amax(1) / 127.0).float()
                codes = torch.round((q / unit.double()[:, None]).float().double()).clamp(-127, 127)
                low, high = cache["low"][at, head].double(), cache["high"][at, head].double()
                whole = torch.maximum(codes[:, None] * low, codes[:, None] * high).sum(2)
                score = ((whole.float() * unit[:, None]) * cache["k_scale"][at, head]).amax(0).tolist()
                forced = {0, n - 1}
                order = sorted(range(n), key=lambda i: (i not in forced, -score[i], i))[:keep]
                lists[t, head, :len(order)] = torch.tensor(sorted(order), dtype=torch.int32)
    return lists
