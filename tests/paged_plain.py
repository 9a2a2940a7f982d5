"""The paged 8-bit cache's operators by their definitions: whole numbers and F32 where the definition rounds to them, 64 bits
elsewhere, a request and a token at a time."""
import numpy as np


def ceil(a, b):
    return -(-a // b)


def plan(before, after, table, ring, counters, page, tokens):
    """The tables as numpy arrays (copied), the rest as lists."""
    table, ring, taken = table.copy(), ring.copy(), ring.copy()
    width, size = table.shape[1], len(ring)
    head, free = int(counters[0]) % size, min(max(int(counters[1]), 0), size)
    left, put = free, 0
    starts, lengths, slots, positions, requests, work = [0], [], [], [], [], []
    for r, (b, a) in enumerate(zip(before, after)):
        b, a = max(int(b), 0), max(int(a), 0)
        have, want = min(ceil(b, page), width), min(ceil(a, page), width)
        for j in range(want, have):
            ring[(head + free + put) % size] = table[r, j]
            put += 1
        n = have
        while n < want and left > 0:
            table[r, n] = taken[(head + free - left) % size]
            left, n = left - 1, n + 1
        length = a if a <= b else min(a, max(b, n * page))
        lengths.append(length)
        for p in range(b, a):
            slots.append(int(table[r, p // page]) * page + p % page if p < length else -1)
            positions.append(p)
            requests.append(r)
        for j in range(b // page, ceil(length, page) if length > b else 0):
            work.append([int(table[r, j]), starts[-1] + max(j * page - b, 0), max(b - j * page, 0), min(length, j * page + page) - max(b, j * page)])
        starts.append(starts[-1] + max(a - b, 0))
    fill = lambda v, n, x: (v + [x] * (n - len(v)))[:n]  # noqa: E731
    items = min(tokens, 2 * len(lengths) + tokens // page)
    return {"table": table, "ring": ring, "starts": starts, "lengths": lengths, "slots": fill(slots, tokens, -1), "positions": fill(positions, tokens, -1),
            "requests": fill(requests, tokens, -1), "work": fill(work, items, [-1, 0, 0, 0]),
            "counters": [(head + free - left) % size, left + put, sum(max(max(int(a), 0) - n, 0) for a, n in zip(after, lengths))]}


def store(cache, k, v, work):
    """cache: numpy arrays, changed in place; k, v float32 [tokens, kv_heads, head_dim]."""
    pages, page = cache["k"].shape[0], cache["k"].shape[2]
    one = np.float32
    for at, row, held, count in work:
        if not (0 <= at < pages and 1 <= count <= page and 0 <= held <= page - count and 0 <= row <= len(k) - count):
            continue
        for name, rows in (("k", k), ("v", v)):
            for h in range(k.shape[1]):
                x = rows[row:row + count, h]
                codes = cache[name][at, h] if name == "k" else cache[name][at, h].T
                size = np.abs(x[np.isfinite(x)]).max(initial=one(0))
                old = cache[name + "_scale"][at, h] if held else one(0)
                with np.errstate(all="ignore"):
                    scale = max(old, one(size) * (one(1) / one(127)))
                    factor = old / scale if held and scale > old else one(1)
                    new = np.rint(x / scale) if scale > 0 else np.zeros_like(x)
                new = np.clip(np.where(np.isnan(new), one(0), new), -127, 127).astype(np.int8)
                again = lambda c: np.rint(c.astype(np.float32) * factor).astype(np.int8)  # noqa: E731
                codes[:held] = again(codes[:held])
                codes[held:held + count] = new
                cache[name + "_scale"][at, h] = scale
                if name == "k" and "low" in cache:
                    for edge, pick in (("low", np.minimum), ("high", np.maximum)):
                        best = pick.reduce(new, axis=0)
                        cache[edge][at, h] = pick(best, again(cache[edge][at, h])) if held else best


def values(cache, at):
    """Pages `at` of the cache as K and V [n, kv_heads, page, head_dim] in 64 bits."""
    k = cache["k"][at].astype(np.float64) * cache["k_scale"][at].astype(np.float64)[..., None, None]
    v = cache["v"][at].astype(np.float64) * cache["v_scale"][at].astype(np.float64)[..., None, None]
    return k, np.swapaxes(v, -1, -2)


def lists(cache, q, table, lengths, starts, keep, first=1, recent=1):
    page, kv_heads, pages = cache["k"].shape[2], cache["k"].shape[1], cache["k"].shape[0]
    group = q.shape[1] // kv_heads
    out = np.full((len(q), kv_heads, keep), -1, dtype=np.int32)
    for r in range(len(lengths)):
        for t in range(starts[r], starts[r + 1]):
            position = lengths[r] - starts[r + 1] + t
            n = position // page + 1 if position >= 0 else 0
            if n == 0:
                continue
            at = table[r, :n]
            at = np.where((at < 0) | (at >= pages), 0, at)
            for h in range(kv_heads):
                x = q[t, h * group:(h + 1) * group].astype(np.float32)
                low, high = cache["low"][at, h].astype(np.float64), cache["high"][at, h].astype(np.float64)
                score = np.full(n, -np.inf, dtype=np.float32)
                with np.errstate(all="ignore"):
                    for row in x:
                        unit = np.float32(np.abs(row).max()) * (np.float32(1) / np.float32(127))
                        if not np.isfinite(unit):
                            continue
                        codes = np.clip(np.rint(row / unit), -127, 127).astype(np.float64) if unit > 0 else np.zeros(len(row))
                        whole = np.where(codes > 0, codes * high, codes * low).sum(1).astype(np.float32)
                        mine = (whole * unit) * cache["k_scale"][at, h]
                        score = np.fmax(score, np.where(np.isnan(mine), np.float32(-np.inf), mine))
                forced = set(range(min(first, n))) | set(range(max(0, n - recent), n))
                order = sorted(range(n), key=lambda j: (j not in forced, -score[j], j))[:keep]
                out[t, h, :len(order)] = sorted(order)
    return out


def attend(cache, q, table, lengths, starts, scale, dtype, window=0, softcap=0.0, sinks=None, picked=None):
    """(values, how far a kernel's may be from them), both [tokens, heads, head_dim] in 64 bits. The distance follows from what
    the operator says of its roundings: a query element is off by half a unit of the row's digits (unit u: its largest magnitude /
    32639, for F32 / 8355711), so a logit by at most scale * u / 2 * sum |k|, and a few units of its own last place (2^-21
    of |s| for three products and a maximum's subtraction); the softcap's slope is at most one, its own error 2^-21 of the cap for
    16-bit rows, 2^-22 for F32; exp and the sums add 2^-20; a probability's F16 is off by 2^-11 of itself (a sum of two F16:
    2^-21) or 2^-25 of the largest weight p * vs, of every token. An error e of every logit moves a sum of p v / sum of p by at most 2 e
    sum p |v|, and the result is rounded to its type (F16's smallest step is 2^-24)."""
    pages, kv_heads, page, d = cache["k"].shape
    heads = q.shape[1]
    group = heads // kv_heads
    out, far = np.zeros(q.shape), np.zeros(q.shape)
    digit = 8355711.0 if dtype == "f32" else 32639.0
    last = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    for r in range(len(lengths)):
        n, length = starts[r + 1] - starts[r], lengths[r]
        at = table[r, :ceil(length, page)]
        there = (at >= 0) & (at < pages)
        k, v = values(cache, np.where(there, at, 0))
        k, v = (np.swapaxes(x, 0, 1).reshape(kv_heads, -1, d)[:, :length] for x in (k, v))
        there = np.repeat(there, page)[:length]
        vs = np.repeat(cache["v_scale"][np.clip(at, 0, pages - 1)].astype(np.float64), page, axis=0)[:length]
        for t in range(n):
            p = length - n + t
            sees = there & (np.arange(length) <= p)
            if window:
                sees &= np.arange(length) > p - window
            for h in range(heads):
                mine = sees
                if picked is not None:
                    chosen = picked[starts[r] + t, h // group]
                    mine = sees & np.isin(np.arange(length) // page, chosen[chosen >= 0])
                if not mine.any():
                    continue
                x, kk, vv = q[starts[r] + t, h].astype(np.float64), k[h // group][mine], v[h // group][mine]
                s = kk @ x * scale
                e = scale * np.abs(x).max() / digit / 2 * np.abs(kk).sum(1).max() + 2.0 ** -21 * np.abs(s).max() + 2.0 ** -20
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                    e += softcap * 2.0 ** (-22 if dtype == "f32" else -21)
                top = max(s.max(), -np.inf if sinks is None else sinks[h])
                w = np.exp(s - top)
                total = w.sum() + (0.0 if sinks is None else np.exp(sinks[h] - top))
                out[starts[r] + t, h] = w @ vv / total
                size = w @ np.abs(vv) / total
                most = np.max(w * vs[mine, h // group]) * 127 * len(s) / total
                far[starts[r] + t, h] = (2 * e + (2.0 ** -21 if dtype == "f32" else 2.0 ** -11)) * size + 2.0 ** -25 * most + last * np.abs(out[starts[r] + t, h])
                if dtype == "f16":
                    far[starts[r] + t, h] += 2.0 ** -25
    return out, far
