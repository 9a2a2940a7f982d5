"""The operators of attention over latent vectors, whose speed is measured: what a program that serves a model with one
shared latent vector a token (keys and values of all heads come from it, a small rotated key beside it) does in a layer.

The paged cache holds, for each token, `width` latent values and `rope` values of the rotated key: both in 16 bits, or the
latent in 8 (E4M3 codes, one E8M0 scale a token). A request's row of the table names its pages in order; a slot is
page * (tokens a page) + offset. A case's "path" says which operator a pass makes:

  rope     part of every head's channels rotated by their token's position: halves or neighbours, plain or YaRN frequencies
  store    new tokens' latent rows (normalised where "norm" says so) and rotated keys into their slots, then slots read back
  project  each head's rows times that head's matrix: queries to the latent width, and values back from it
  attend   the absorbed form: queries of the latent width over the cache's pages, causal, any number of new tokens a request
  prompt   the expanded form: keys and values of every head, one rotated key for all of them, causal, ragged
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
BASE, EPS = 10000.0, 1e-6


def listed():
    return [
        # The smallest calls: a decode step of 64 requests, the last 64 channels of each head's query rotated, positions far apart.
        {"name": "rope_64_tokens", "path": "rope", "tokens": 64, "heads": 32, "head_dim": 192, "first": 128, "n_dims": 64, "layout": "interleaved",
         "yarn": True, "dtype": "bf16", "longest": 131072},
        # A prompt's queries, whole heads rotated.
        {"name": "rope_prompt_8192", "path": "rope", "tokens": 8192, "heads": 32, "head_dim": 128, "first": 0, "n_dims": 128, "layout": "half",
         "yarn": False, "dtype": "bf16", "longest": 8192},
        # A decode step's rows of 64 requests into an 8-bit cache and back.
        {"name": "store_64_tokens", "path": "store", "requests": 64, "page": 64, "longest": 8192, "fresh": 1, "width": 512, "rope": 64, "bits": 8,
         "norm": False, "read": "new", "layout": "interleaved", "dtype": "bf16", "kept": "bf16"},
        # Prompts behind cached beginnings: their rows normalised and stored, then all the request's rows read for the expanded form.
        {"name": "store_prompts", "path": "store", "requests": 5, "page": 16, "longest": 6000, "fresh": 2000, "width": 512, "rope": 64, "bits": 16,
         "norm": True, "read": "held", "layout": "interleaved", "dtype": "f32", "kept": "bf16"},
        # A decode step's queries to the latent width: the matrices of 128 heads are what is read.
        {"name": "project_64_tokens", "path": "project", "tokens": 64, "heads": 128, "k": 128, "n": 512, "dtype": "bf16"},
        # A prompt chunk's values back from it, an odd number of rows.
        {"name": "project_2001_tokens", "path": "project", "tokens": 2001, "heads": 32, "k": 512, "n": 128, "dtype": "bf16"},
        # One request's decode step, a shard of 16 heads: latency.
        {"name": "attend_1_request_2000", "path": "attend", "requests": 1, "page": 64, "longest": 2000, "fresh": 1, "heads": 16, "width": 512, "rope": 64,
         "bits": 16, "dtype": "bf16"},
        # A full server's decode step on such a shard, an 8-bit cache.
        {"name": "attend_64_requests_8_bit", "path": "attend", "requests": 64, "page": 64, "longest": 16384, "fresh": 1, "heads": 16, "width": 512,
         "rope": 64, "bits": 8, "dtype": "bf16"},
        # The same with all 128 heads on the card: the matrix products and the cache's bytes take about as long.
        {"name": "attend_48_requests_128_heads", "path": "attend", "requests": 48, "page": 64, "longest": 8192, "fresh": 1, "heads": 128, "width": 512,
         "rope": 64, "bits": 16, "dtype": "bf16"},
        # Chunks of prompts of no round length behind cached beginnings, 16-token pages, the smaller widths.
        {"name": "attend_chunks", "path": "attend", "requests": 3, "page": 16, "longest": 5000, "fresh": 300, "heads": 20, "width": 256, "rope": 32,
         "bits": 16, "dtype": "f16"},
        # A prompt in the expanded form: the largest.
        {"name": "prompt_4096", "path": "prompt", "requests": 1, "longest": 4096, "fresh": 4096, "heads": 32, "nope": 128, "rope": 64, "value": 128,
         "dtype": "bf16"},
        # Ragged prompts behind keys of earlier chunks, the smaller heads.
        {"name": "prompt_ragged", "path": "prompt", "requests": 6, "longest": 3500, "fresh": 700, "heads": 12, "nope": 64, "rope": 32, "value": 64,
         "dtype": "f16"},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    path = rng.choice(["rope", "store", "project", "attend", "attend", "attend", "prompt", "prompt"])
    narrow = rng.choice(["bf16", "f16"])
    layout = rng.choice(["half", "interleaved"])
    if path == "rope":
        heads = rng.choice([1, 8, 20, 32, 64, 128])
        head_dim, first, n_dims = rng.choice([(128, 0, 128), (192, 128, 64), (80, 48, 32), (64, 0, 64), (128, 0, 64), (256, 0, 128)])
        return {"path": path, "tokens": _log(rng, 1, min(8192, (1 << 25) // (heads * head_dim))), "heads": heads, "head_dim": head_dim, "first": first,
                "n_dims": n_dims, "layout": layout, "yarn": rng.random() < 0.5, "dtype": rng.choice(list(DTYPES)), "longest": _log(rng, 16, 1000000)}
    width, rope = rng.choice([(512, 64), (512, 64), (256, 32), (256, 64), (512, 32)])
    page = rng.choice([16, 32, 64, 128])
    if path == "store":
        fresh = rng.choice([1, _log(rng, 2, 2000)])
        bits = rng.choice([8, 16])
        return {"path": path, "requests": _log(rng, 1, 64 if fresh == 1 else 7), "page": page, "longest": max(fresh, _log(rng, 16, 6000)), "fresh": fresh,
                "width": width, "rope": rope, "bits": bits, "norm": bits == 16 and rng.random() < 0.5, "read": rng.choice(["new", "held"]),
                "layout": layout, "dtype": rng.choice(list(DTYPES)), "kept": narrow}
    if path == "project":
        k, n = rng.choice([(128, 512), (512, 128), (64, 256), (256, 64), (128, 256)])
        return {"path": path, "tokens": _log(rng, 1, 2048), "heads": rng.choice([8, 12, 16, 20, 32]), "k": k, "n": n, "dtype": narrow}
    if path == "attend":
        base = {"heads": rng.choice([8, 16, 20, 32, 64, 128]), "width": width, "rope": rope, "bits": rng.choice([8, 16]), "dtype": narrow}
        if rng.random() < 0.7:
            requests = _log(rng, 1, 64)
            return {"path": path, "requests": requests, "page": page, "longest": _log(rng, 8, min(100000, 300000 // requests)),
                    "fresh": rng.choice([1, 1, _log(rng, 2, 4)]), **base}
        requests = _log(rng, 1, 4)
        fresh = _log(rng, 5, 300)
        return {"path": path, "requests": requests, "page": page, "longest": max(fresh, _log(rng, 16, 5000)), "fresh": fresh,
                **{**base, "heads": min(base["heads"], 32)}}
    requests = _log(rng, 1, 6)
    nope, rope, value, heads = rng.choice([(128, 64, 128, 8), (128, 64, 128, 32), (64, 32, 64, 12), (64, 64, 128, 20), (128, 32, 64, 5)])
    fresh = _log(rng, 1, 2000)
    return {"path": path, "requests": requests, "longest": max(fresh, _log(rng, 16, 4000)), "fresh": fresh, "heads": heads, "nope": nope, "rope": rope,
            "value": value, "dtype": narrow}


# ---------------------------------------------------------------- inputs


def _requests(case):
    """(before, after) of every request: the first is the longest and has the most new tokens, the others' are spread over
    their ranges' logarithms. With five or more the last one has nothing new."""
    rng = random.Random(case["requests"] * 1000003 + case["longest"] * 1009 + case["fresh"])
    before, after = [], []
    for r in range(case["requests"]):
        length = case["longest"] if r == 0 else _log(rng, max(1, case["longest"] // 8), case["longest"])
        new = case["fresh"] if r == 0 or case["fresh"] == 1 else _log(rng, 1, case["fresh"])
        new = min(new, length)
        if r == case["requests"] - 1 and case["requests"] >= 5:
            new = 0
        before.append(length - new), after.append(length)
    return before, after


def _starts(counts):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _corrections(n_dims):
    """YaRN's first and last mixed pair: 32 turns and one turn over 4096 original positions."""
    at = [n_dims * math.log(4096.0 / (turns * 2.0 * math.pi)) / (2.0 * math.log(BASE)) for turns in (32.0, 1.0)]
    return max(0.0, math.floor(at[0])), min(n_dims - 1.0, math.ceil(at[1]))


def _rope_options(case):
    if not case.get("yarn"):
        return {}
    return {"freq_scale": 1.0 / 40.0, "ext_factor": 1.0, "corr_dims": _corrections(case["n_dims"])}


def _codes(x):
    """E4M3 codes of float32 rows (nearest, ties to even, at most 448) and the rows' E8M0 scales."""
    bits = (x.abs().amax(-1) * (1.0 / 448.0)).view(torch.int32)
    e = ((bits >> 23) + ((bits & 0x7FFFFF) != 0).to(torch.int32)).clamp(max=253)
    y = x * ((254 - e) << 23).view(torch.float32)[..., None]
    bits = y.abs().contiguous().view(torch.int32)
    large = ((bits + 0x7FFFF + ((bits >> 20) & 1)) >> 20) - 960
    small = torch.round(y.abs() * 512.0).to(torch.int32)
    code = torch.where(bits < 0x3C800000, small, large).clamp(max=0x7E) + torch.where(y < 0, 128, 0)
    return code.to(torch.uint8), e.to(torch.uint8)


def _values(codes, scales, dtype):
    """What codes and scales stand for, in `dtype` (32 or 64 bits; exactly)."""
    c = codes.to(torch.int32)
    mag, sign = c & 0x7F, 1 - 2 * (c >> 7)
    exponent = (mag >> 3).clamp(min=1)
    fraction = torch.where(mag < 8, mag, 8 + (mag & 7))
    x = torch.ldexp((fraction * sign).to(dtype), exponent - 10)
    return torch.ldexp(x, (scales.to(torch.int32) - 127)[..., None])


def _cache(case, pages, g, kept):
    """Latent rows as a normalisation leaves them, keys of the same size; neighbouring tokens' share a direction."""
    page, width, rope = case["page"], case["width"], case["rope"]
    step = max(1, (1 << 26) // (page * width))
    bits8 = case["bits"] == 8
    latent = torch.empty((pages, page, width), dtype=torch.uint8 if bits8 else kept, device="cuda")
    scale = torch.empty((pages, page), dtype=torch.uint8, device="cuda") if bits8 else None
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = torch.randn((n, page, width), device="cuda", generator=g) + 0.7 * torch.randn((n, 1, width), device="cuda", generator=g)
        if bits8:
            latent[at:at + n], scale[at:at + n] = _codes(x)
        else:
            latent[at:at + n] = x.to(kept)
    key = torch.randn((pages, page, rope), device="cuda", generator=g).to(kept)
    return {"latent": latent, "rope": key, **({"scale": scale} if bits8 else {})}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if own and case["path"] in ("rope", "store"):
        from llmp_amd import ops
        s["turns"] = ops.rope_table(case["n_dims"] if case["path"] == "rope" else case["rope"], BASE, **_rope_options(case))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, size=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * size).to(dtype)

    if case["path"] == "rope":
        tokens, longest = case["tokens"], case["longest"]
        s["x"] = normal(tokens, case["heads"], case["head_dim"])
        s["positions"] = torch.randint(0, longest, (tokens,), device="cuda", generator=g).to(torch.int32)
        if tokens == longest:  # one prompt
            s["positions"] = torch.arange(tokens, dtype=torch.int32, device="cuda")
        return s
    if case["path"] == "project":
        s["x"] = normal(case["tokens"], case["heads"], case["k"])
        s["w"] = normal(case["heads"], case["n"], case["k"], size=1.0 / math.sqrt(case["k"]))
        return s
    before, after = _requests(case)
    fresh = [a - b for b, a in zip(before, after)]
    starts = _starts(fresh)
    tokens = starts[-1]
    s["tokens"], s["most"], s["starts"] = tokens, max(1, max(fresh)), _ints(starts)
    s["before"], s["lengths"] = _ints(before), _ints(after)
    if case["path"] == "prompt":
        key_starts = _starts(after)
        keys, heads = key_starts[-1], case["heads"]
        s["key_starts"] = _ints(key_starts)
        s["scale"] = 1.0 / math.sqrt(case["nope"] + case["rope"])
        s["q"] = normal(tokens, heads, case["nope"] + case["rope"], size=1.5)
        # A product's rows: every head's key and value side by side, as the expansion of the latent rows leaves them.
        s["kv"] = normal(keys, heads, case["nope"] + case["value"])
        s["k_rope"] = normal(keys, case["rope"])
        return s
    page, kept = case["page"], DTYPES[case.get("kept", case["dtype"])]
    held = [-(-a // page) for a in after]
    pages, width = sum(held) + 1, max(held) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    counts = torch.tensor(held, device="cuda")
    ends = torch.cumsum(counts, 0)
    column = torch.arange(width, device="cuda")
    place = (ends - counts)[:, None] + column
    s["table"] = torch.where(column < counts[:, None], order[place.clamp(max=pages - 1)], torch.full_like(order[:1], -1)).contiguous()
    s["cache"] = _cache(case, pages, g, kept)
    if case["path"] == "attend":
        s["q_latent"] = normal(tokens, case["heads"], case["width"], size=1.0)
        s["q_rope"] = normal(tokens, case["heads"], case["rope"], size=1.0)
        s["scale"] = 2.0 / math.sqrt(case["width"] + case["rope"])
        return s
    request = torch.repeat_interleave(torch.arange(case["requests"], device="cuda"), torch.tensor(fresh, device="cuda"))
    position = torch.arange(tokens, device="cuda") - s["starts"][request] + s["before"][request]
    s["positions"] = position.to(torch.int32)
    s["slots"] = (s["table"][request, position // page] * page + position % page).to(torch.int32)
    s["read_slots"] = s["slots"]
    if case["read"] == "held":
        request = torch.repeat_interleave(torch.arange(case["requests"], device="cuda"), torch.tensor(after, device="cuda"))
        position = torch.arange(sum(after), device="cuda") - torch.tensor(_starts(after), device="cuda")[request]
        s["read_slots"] = (s["table"][request, position // page] * page + position % page).to(torch.int32)
    # The down projection's rows: the latent's values, then the key's.
    s["rows"] = normal(tokens, case["width"] + case["rope"]) * torch.exp(0.5 * torch.randn(case["width"] + case["rope"], device="cuda", generator=g)).to(dtype)
    s["weight"] = 1.0 + 0.2 * torch.randn(case["width"], device="cuda", generator=g) if case["norm"] else None
    return s


# ---------------------------------------------------------------- the passes


def run(s):
    if own:
        return _own(s)
    return {"rope": _rope, "store": _store, "project": _project, "attend": _attend, "prompt": _prompt}[s["path"]](s)


def _own(s):
    from llmp_amd import ops
    if s["path"] == "rope":
        return {"y": ops.rope(s["x"], s["positions"], s["turns"], layout=s["layout"], first=s["first"])}
    if s["path"] == "project":
        return {"y": ops.latent_project(s["x"], s["w"])}
    if s["path"] == "prompt":
        k, v = s["kv"][..., :s["nope"]], s["kv"][..., s["nope"]:]
        return {"out": ops.latent_prompt(s["q"], k, s["k_rope"], v, s["starts"], s["scale"], key_starts=s["key_starts"], most=s["most"])}
    cache = s["cache"]
    if s["path"] == "attend":
        return {"out": ops.latent_attend(cache, s["q_latent"], s["q_rope"], s["table"], s["lengths"], s["starts"], s["scale"], most=s["most"])}
    ops.latent_store(cache, s["rows"][:, :s["width"]], s["rows"][:, s["width"]:], s["slots"], s["positions"], s["turns"], layout=s["layout"],
                     weight=s["weight"], eps=EPS)
    latent, rope = ops.latent_read(cache, s["read_slots"])
    return {"latent": latent, "rope": rope}


def _rotate(x, positions, n_dims, layout, options):
    """The last axis (n_dims channels) of x [tokens, ..., n_dims] rotated; angles in 64 bits, values in 32."""
    pair = torch.arange(n_dims // 2, dtype=torch.float64, device=x.device)
    frequency = BASE ** (-2.0 * pair / n_dims)
    size = 1.0
    if options:
        low, high = options["corr_dims"]
        mix = 1.0 - ((pair - low) / max(0.001, high - low)).clamp(0.0, 1.0)
        frequency = frequency * (options["freq_scale"] * (1.0 - mix) + mix)
        size = 1.0 + 0.1 * math.log(1.0 / options["freq_scale"])
    angle = positions.double()[:, None] * frequency
    shape = (x.shape[0],) + (1,) * (x.dim() - 2) + (n_dims // 2,)
    cos, sin = ((f(angle) * size).float().view(shape) for f in (torch.cos, torch.sin))
    x = x.float()
    if layout == "half":
        a, b = x[..., :n_dims // 2], x[..., n_dims // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _rope(s):
    x, first, n = s["x"], s["first"], s["n_dims"]
    turned = _rotate(x[..., first:first + n], s["positions"], n, s["layout"], _rope_options(s))
    return {"y": torch.cat([x[..., :first], turned.to(x.dtype), x[..., first + n:]], -1)}


def _store(s):
    cache, width, page = s["cache"], s["width"], s["page"]
    kept = cache["rope"].dtype
    x = s["rows"][:, :width].float()
    if s["weight"] is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"]
    key = _rotate(s["rows"][:, width:], s["positions"], s["rope"], s["layout"], {})
    slots, read = s["slots"].long(), s["read_slots"].long()
    flat = {name: c.flatten(0, 1) for name, c in cache.items()}
    flat["rope"][slots] = key.to(kept)
    if s["bits"] == 8:
        flat["latent"][slots], flat["scale"][slots] = _codes(x)
        return {"latent": _values(flat["latent"][read], flat["scale"][read], torch.float32).to(kept), "rope": flat["rope"][read]}
    flat["latent"][slots] = x.to(kept)
    return {"latent": flat["latent"][read], "rope": flat["rope"][read]}


def _project(s):
    x, w = s["x"].float(), s["w"].float()
    y = torch.matmul(x.transpose(0, 1).contiguous(), w.transpose(1, 2).contiguous())
    return {"y": y.transpose(0, 1).to(s["x"].dtype).contiguous()}


def _softmax(score, hidden):
    score = score.masked_fill(hidden, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _attend(s):
    cache, page = s["cache"], s["page"]
    q = torch.cat([s["q_latent"], s["q_rope"]], -1).float()
    out = torch.zeros(s["q_latent"].shape, dtype=torch.float32, device=q.device)
    before, after = _requests(s)
    start = 0
    for r, (b, a) in enumerate(zip(before, after)):
        n = a - b
        if n:
            at = s["table"][r, :-(-a // page)].long()
            c = _values(cache["latent"][at], cache["scale"][at], torch.float32) if "scale" in cache else cache["latent"][at].float()
            c = c.reshape(-1, s["width"])[:a]
            k = torch.cat([c, cache["rope"][at].float().reshape(-1, s["rope"])[:a]], 1)
            score = torch.matmul(q[start:start + n].reshape(n * s["heads"], -1), k.T.contiguous()).view(n, s["heads"], a) * s["scale"]
            j = torch.arange(a, device=q.device)
            p = _softmax(score, (j > torch.arange(b, a, device=q.device)[:, None])[:, None, :])
            out[start:start + n] = torch.matmul(p.view(n * s["heads"], a), c).view(n, s["heads"], -1)
        start += n
    return {"out": out.to(s["q_latent"].dtype)}


def _prompt(s):
    q, kv, k_rope = s["q"].float(), s["kv"].float(), s["k_rope"].float()
    heads, nope = s["heads"], s["nope"]
    out = torch.zeros((s["tokens"], heads, s["value"]), dtype=torch.float32, device=q.device)
    before, after = _requests(s)
    start = key = 0
    for b, a in zip(before, after):
        n = a - b
        if n:
            x = q[start:start + n].transpose(0, 1).contiguous()
            k = torch.cat([kv[key:key + a, :, :nope], k_rope[key:key + a, None, :].expand(-1, heads, -1)], -1)
            score = torch.matmul(x, k.permute(1, 2, 0).contiguous()) * s["scale"]
            j = torch.arange(a, device=q.device)
            p = _softmax(score, j > torch.arange(b, a, device=q.device)[:, None])
            out[start:start + n] = torch.matmul(p, kv[key:key + a, :, nope:].transpose(0, 1).contiguous()).transpose(0, 1)
        start, key = start + n, key + a
    return {"out": out.to(s["q"].dtype)}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    size = SIZES[case["dtype"]]
    if case["path"] == "rope":
        rows = case["tokens"] * case["heads"]
        return {"bytes": 2 * rows * case["head_dim"] * size + 4 * case["tokens"] + 4 * case["n_dims"], "flops": 3 * rows * case["n_dims"]}
    if case["path"] == "project":
        t, h, k, n = case["tokens"], case["heads"], case["k"], case["n"]
        return {"bytes": size * h * (t * (k + n) + k * n), "flops": 2 * t * h * k * n}
    before, after = _requests(case)
    fresh = [a - b for b, a in zip(before, after)]
    tokens = sum(fresh)
    pairs = sum((b + 1 + a) * (a - b) // 2 for b, a in zip(before, after))
    seen = sum(a for a, n in zip(after, fresh) if n)
    if case["path"] == "prompt":
        heads, nope, rope, value = case["heads"], case["nope"], case["rope"], case["value"]
        return {"bytes": size * (tokens * heads * (nope + rope + value) + seen * (heads * (nope + value) + rope)),
                "flops": 2 * pairs * heads * (nope + rope + value)}
    width, rope = case["width"], case["rope"]
    kept = SIZES[case.get("kept", case["dtype"])]
    row = (width + 1 if case["bits"] == 8 else kept * width) + kept * rope  # a token's in the cache
    if case["path"] == "store":
        read = tokens if case["read"] == "new" else sum(after)
        # Rows in and into the cache with their slots and positions; rows out of the cache as values.
        return {"bytes": tokens * (size * (width + rope) + row + 8) + read * (row + kept * (width + rope) + 4) + (4 * width if case["norm"] else 0),
                "flops": 4 * tokens * (width + rope)}
    return {"bytes": seen * row + size * tokens * case["heads"] * (2 * width + rope) + 4 * (seen // case["page"]),
            "flops": 2 * pairs * case["heads"] * (2 * width + rope)}


# ---------------------------------------------------------------- the definitions, in 64 bits


def _exact_rotation(x, positions, layout, options):
    """Pair by pair as a complex number turned."""
    n = x.shape[-1]
    x = x.double()
    parts = []
    for p in range(n // 2):
        f = math.exp(-2.0 * p / n * math.log(BASE))
        size = 1.0
        if options:
            low, high = options["corr_dims"]
            keep = 1.0 - min(1.0, max(0.0, (p - low) / max(0.001, high - low)))
            f = f * options["freq_scale"] * (1.0 - keep) + f * keep
            size = 1.0 - 0.1 * math.log(options["freq_scale"])
        i, j = (p, p + n // 2) if layout == "half" else (2 * p, 2 * p + 1)
        angle = positions.double() * f
        turn = torch.polar(torch.full_like(angle, size), angle).view((-1,) + (1,) * (x.dim() - 2))
        parts.append((i, j, torch.complex(x[..., i].contiguous(), x[..., j].contiguous()) * turn))
    y = torch.empty_like(x)
    for i, j, z in parts:
        y[..., i], y[..., j] = z.real, z.imag
    return y


def _exact_codes(x):
    """The values that 8 bits hold of x: the smallest power of two s with |x| <= 448 s, then the nearest E4M3 value."""
    most = x.abs().amax(-1, keepdim=True)
    s = torch.exp2(torch.ceil(torch.log2(most / 448.0)).clamp(min=-127.0))
    s = torch.where(most > 448.0 * s, 2.0 * s, s)
    s = torch.where((most <= 224.0 * s) & (s > 2.0 ** -127), 0.5 * s, s)
    y = x / s
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(y / step) * step * s


def exact(case, seed):
    s = prepare(case, seed)
    if case["path"] == "rope":
        y, first, n = s["x"].double(), case["first"], case["n_dims"]
        y[..., first:first + n] = _exact_rotation(s["x"][..., first:first + n], s["positions"], case["layout"], _rope_options(case))
        return {"y": y}
    if case["path"] == "project":
        y = torch.empty((case["tokens"], case["heads"], case["n"]), dtype=torch.float64, device=s["x"].device)
        for h in range(case["heads"]):
            y[:, h] = torch.mm(s["x"][:, h].double(), s["w"][h].double().T.contiguous())
        return {"y": y}
    if case["path"] == "store":
        return _exact_store(s)
    starts = s["starts"].tolist()
    lengths = s["lengths"].tolist()
    value = case["width"] if case["path"] == "attend" else case["value"]
    out = torch.zeros((s["tokens"], case["heads"], value), dtype=torch.float64, device=s["starts"].device)
    key = 0
    for r, length in enumerate(lengths):
        n = starts[r + 1] - starts[r]
        if n and case["path"] == "attend":
            j = torch.arange(length, device=out.device)
            at, offset = s["table"][r].long()[j // case["page"]], j % case["page"]
            c = s["cache"]["latent"][at, offset]
            c = _values(c, s["cache"]["scale"][at, offset], torch.float64) if case["bits"] == 8 else c.double()
            k = s["cache"]["rope"][at, offset].double().T.contiguous()
            step = max(1, (1 << 27) // (length * case["heads"]))
            for t0 in range(0, n, step):
                t1 = min(n, t0 + step)
                rows = slice(starts[r] + t0, starts[r] + t1)
                m = (t1 - t0) * case["heads"]
                score = torch.mm(s["q_latent"][rows].double().reshape(m, -1), c.T.contiguous()) + torch.mm(s["q_rope"][rows].double().reshape(m, -1), k)
                out[rows] = torch.mm(_exact_weights(score, s["scale"], length - n + t0, case["heads"]), c).view(t1 - t0, case["heads"], value)
        elif n:
            shared = s["k_rope"][key:key + length].double().T.contiguous()
            for h in range(case["heads"]):
                q = s["q"][starts[r]:starts[r + 1], h].double()
                kv = s["kv"][key:key + length, h].double()
                score = torch.mm(q[:, :case["nope"]].contiguous(), kv[:, :case["nope"]].T.contiguous()) + torch.mm(q[:, case["nope"]:].contiguous(), shared)
                out[starts[r]:starts[r + 1], h] = torch.mm(_exact_weights(score, s["scale"], length - n, 1), kv[:, case["nope"]:].contiguous())
        key += length
    return {"out": out}


def _exact_weights(score, scale, first, heads):
    """Softmax over the positions that each row sees; row i is of the token at position first + i // heads."""
    row = first + torch.div(torch.arange(score.shape[0], device=score.device), heads, rounding_mode="floor")
    j = torch.arange(score.shape[1], device=score.device)
    return torch.softmax(torch.where(j <= row[:, None], score * scale, -math.inf), 1)


def _exact_store(s):
    cache, width = s["cache"], s["width"]
    x = s["rows"][:, :width].double()
    if s["weight"] is not None:
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / width + EPS) * s["weight"].double()
    if s["bits"] == 8:
        x = _exact_codes(x)
    key = _exact_rotation(s["rows"][:, width:], s["positions"], s["layout"], {})
    latent = cache["latent"].view(-1, width)
    latent = _values(latent, cache["scale"].view(-1), torch.float64) if s["bits"] == 8 else latent.double()
    rope = cache["rope"].view(-1, s["rope"]).double()
    latent[s["slots"].long()] = x
    rope[s["slots"].long()] = key
    read = s["read_slots"].long()
    return {"latent": latent[read], "rope": rope[read]}
