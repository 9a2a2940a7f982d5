"""The paged 8-bit KV cache on the device (llmp_hip_paged_*) against its operators' definitions in tests/paged_plain.py: the
plan, the store and the selection bit for bit, the attention within the distance that its stated roundings give."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import paged_plain as plain
from llmp_amd import _lib, ops, synth

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def dev(a, device):
    return torch.from_numpy(np.ascontiguousarray(a)).to(device)


def rounded(x, dtype):
    """x as values of the type, and as floats again."""
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(TYPES[dtype])
    return t, t.float().numpy()


def same(got, want, name):
    got, want = got.cpu().numpy() if isinstance(got, torch.Tensor) else got, np.asarray(want)
    wrong = np.argwhere(~((got == want) | ((got != got) & (want != want)))) if got.shape == want.shape else None
    if wrong is None or len(wrong):
        pytest.fail(f"{name}: shapes {got.shape}, {want.shape}" if wrong is None else
                    f"{name}: {len(wrong)} of {want.size} differ, the first at {wrong[:4].tolist()}: {got[tuple(wrong[0])]}, not {want[tuple(wrong[0])]}")


# ---------------------------------------------------------------- the plan


def check_plan(device, before, after, table, ring, counters, page, tokens, in_place=False):
    want = plain.plan(before, after, table, ring, counters, page, tokens)
    t, r, c = dev(table, device), dev(ring, device), dev(np.asarray(counters, dtype=np.int32), device)
    out = None
    if in_place:
        n = len(before)
        out = {k: torch.empty(s, dtype=torch.int32, device=device) for k, s in
               {"work": (len(want["work"]), 4), "slots": tokens, "positions": tokens, "requests": tokens, "starts": n + 1, "lengths": n}.items()}
        out["counters"] = c
    got = ops.paged_plan(dev(before, device), dev(after, device), t, r, c, page, tokens, out=out)
    same(t, want["table"], "table")
    same(r, want["ring"], "ring")
    for name in ("starts", "lengths", "slots", "positions", "requests", "counters"):
        same(got[name], np.asarray(want[name], dtype=np.int32), name)
    same(got["work"], np.asarray(want["work"], dtype=np.int32).reshape(-1, 4), "work")
    return want


@pytest.mark.parametrize("requests,page,width,most", [(1, 16, 9, 40), (5, 64, 7, 200), (64, 64, 40, 3), (77, 16, 50, 90), (1000, 32, 12, 60),
                                                      (1024, 16, 30, 7), (1025, 48, 9, 9), (2500, 16, 20, 40)])
def test_steps_of_requests_that_grow_shrink_and_end(device, requests, page, width, most):
    """Steps on end from an empty cache, until the ring has gone round and, in some of them, run out."""
    g = np.random.default_rng(requests * page + most)
    pages = max(3, requests * width // 4)
    table = np.full((requests, width), -1, dtype=np.int32)
    ring = g.permutation(pages).astype(np.int32)
    counters = [int(g.integers(pages)), pages, 0]
    ring = np.roll(ring, counters[0])
    held = np.zeros(requests, dtype=np.int32)
    short = 0
    for step in range(6):
        grow = g.integers(0, most + 1, requests) * (g.random(requests) < 0.7)
        after = np.where(g.random(requests) < 0.15, g.integers(0, held + 1), np.minimum(held + grow, width * page)).astype(np.int32)
        fresh = int(np.maximum(after - held, 0).sum())
        want = check_plan(device, held, after, table, ring, counters, page, fresh + step, in_place=step % 2 == 1)
        table, ring, counters = want["table"], want["ring"], want["counters"]
        held = np.asarray(want["lengths"], dtype=np.int32)
        short += counters[2]
        counters = counters[:2] + [0]
        owned = [int(table[r, j]) for r in range(requests) for j in range(plain.ceil(int(held[r]), page))]
        free = [int(ring[(counters[0] + i) % pages]) for i in range(counters[1])]
        assert sorted(owned + free) == list(range(pages))  # every page has one owner
    assert requests != 1000 or short > 0  # (the case that runs out of pages)


def test_plan_lengths_out_of_range_and_no_tokens(device):
    table = np.arange(12, dtype=np.int32).reshape(3, 4)
    ring = np.arange(100, 108, dtype=np.int32)
    # Negative lengths count as zero, a request stops at its table's width, a count past the ring at the ring.
    check_plan(device, np.array([-5, 30, 64], np.int32), np.array([20, 500, 64], np.int32), table, ring, [7, 8, 0], 16, 600)
    check_plan(device, np.array([3, 9, 0], np.int32), np.array([3, 0, 0], np.int32), table, ring, [-3, 4, 0], 16, 0)
    check_plan(device, np.array([3, 9, 0], np.int32), np.array([5, 11, 1], np.int32), table, ring, [2, 0, 0], 16, 2)  # fewer rows than tokens


# ---------------------------------------------------------------- the store


def random_cache(g, pages, kv_heads, page, d, edges=True):
    cache = {"k": g.integers(-127, 128, (pages, kv_heads, page, d)).astype(np.int8), "v": g.integers(-127, 128, (pages, kv_heads, d, page)).astype(np.int8)}
    for name in ("k", "v"):
        cache[name + "_scale"] = (g.random((pages, kv_heads)) * 0.02 + 0.01).astype(np.float32)
    if edges:
        cache["low"], cache["high"] = cache["k"].min(2), cache["k"].max(2)
    return cache


def to_device(cache, device):
    return {k: dev(v, device) for k, v in cache.items()}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kv_heads,page,d", [(1, 16, 64), (3, 64, 128), (2, 48, 256), (2, 256, 256), (8, 128, 64)])
def test_store_and_read_are_their_definition_bit_for_bit(device, dtype, kv_heads, page, d):
    g = np.random.default_rng(page + d + kv_heads)
    pages = 11
    cache = random_cache(g, pages, kv_heads, page, d)
    # Whole pages, single tokens at a page's start, middle and end, a page's rest, an odd run inside; and items that do not fit.
    work, row = [], 0
    for at, held, count in [(3, 0, page), (0, 0, 1), (7, page - 1, 1), (9, 5, 1), (1, 3, page - 3), (5, 7, 6), (2, 0, 13), (10, 9, 5)]:
        work.append([at, row, held, count])
        row += count
    bad = [[-1, 0, 0, 0], [4, 0, 0, 0], [pages, 0, 0, 1], [4, row, 0, 1], [4, 0, page, 1], [4, 0, -1, 2], [4, -1, 0, 1], [4, 0, 1, page], [6, row - 1, 0, 2]]
    work = np.array(work[:4] + bad + work[4:], dtype=np.int32)
    size = np.array([0.3, 5.0, 0.2, 1.0, 2.5, 0.01, 1.0, 0.0], dtype=np.float32)  # some scales rise, some do not; one run is zeros
    rows = [g.standard_normal((row, kv_heads, d), dtype=np.float32) for _ in range(2)]
    for x in rows:
        for (at, first, held, count), s in zip([w for w in work.tolist() if w not in bad], size):
            x[first:first + count] *= s
    rows[0][2:6, 0, 3], rows[0][page, 0, 0], rows[1][3, 0, 5], rows[1][1, 0, 0] = np.inf, np.nan, -np.inf, np.nan
    (kt, k), (vt, v) = rounded(rows[0], dtype), rounded(rows[1], dtype)
    on_device = to_device(cache, device)
    # Strided rows: K and V side by side, as one product leaves them.
    both = torch.cat([kt, torch.zeros_like(kt[:, :1]), vt], 1).to(device)
    ops.paged_store(on_device, both[:, :kv_heads], both[:, kv_heads + 1:], dev(work, device))
    plain.store(cache, k, v, work.tolist())
    for name in cache:
        same(on_device[name], cache[name], name)
    asked = np.array([3, -1, 10, pages, 0, 0, 7], dtype=np.int32)
    for out in TYPES:
        got = ops.paged_read(on_device, dev(np.stack([asked, asked * 0 + 99], 1), device)[:, 0], TYPES[out])
        inside = (asked >= 0) & (asked < pages)
        for x, codes, scale in zip(got, (cache["k"], np.swapaxes(cache["v"], 2, 3)), (cache["k_scale"], cache["v_scale"])):
            at = np.where(inside, asked, 0)
            want = np.where(inside[:, None, None, None], codes[at].astype(np.float32) * scale[at][..., None, None], np.float32(0))
            same(x.float(), rounded(want, out)[1], f"read {out}")


def test_store_without_edges_and_a_page_filled_token_by_token(device):
    """One token at a time, growing: every step may raise the scale and round what is held again."""
    g = np.random.default_rng(5)
    cache = random_cache(g, 3, 2, 32, 64, edges=False)
    on_device = to_device(cache, device)
    x = (g.standard_normal((2, 32, 2, 64)) * np.linspace(0.1, 3.0, 32)[None, :, None, None]).astype(np.float32)
    k, v = dev(x[0], device), dev(x[1], device)
    for t in range(32):
        ops.paged_store(on_device, k, v, dev(np.array([[1, t, t, 1]], dtype=np.int32), device))
        plain.store(cache, x[0], x[1], [[1, t, t, 1]])
        for name in cache:
            same(on_device[name], cache[name], f"{name} at {t}")
    err = np.abs(plain.values(cache, [1])[0][0] - np.swapaxes(x[0], 0, 1))
    assert err.max() <= cache["k_scale"][1].max() * 3  # (a code rounded again and again drifts by less than a few steps)


# ---------------------------------------------------------------- attention


def serving(g, lengths, fresh, kv_heads, page, d, spare=3):
    """A cache with the requests' pages in a random order, everything that no token lies in spoiled: codes any, scales NaN, table
    entries past a request's pages any number."""
    width = max(1, max(plain.ceil(n, page) for n in lengths)) + 1
    need = [plain.ceil(n, page) for n in lengths]
    pages = sum(need) + spare
    cache = random_cache(g, pages, kv_heads, page, d)
    order = g.permutation(pages)
    table = g.choice(np.array([-1, -7, pages, 1 << 30, 0], dtype=np.int32), (len(lengths), width))
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    for name in ("k_scale", "v_scale"):
        cache[name][order[at:]] = np.nan
    starts = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
    return cache, table, np.asarray(lengths, dtype=np.int32), starts


def widened(table, cache, tokens, most, heads):
    """The table with as many more columns, of any entries, as make a call of rows for it one of the prompts' form (rows times the
    tokens a table row can name times head size: llmp_amd/csrc/paged_attend.hip, kFewWork)."""
    pages, kv_heads, page, d = cache["k"].shape
    if most * heads // kv_heads <= 64:
        return table
    more = 4000000 * 128 // (tokens * heads // kv_heads * d * page) + 2
    spoiled = np.random.default_rng(5).choice(np.array([-1, -7, pages, 1 << 30, 0], dtype=np.int32), (len(table), more))
    return np.concatenate([table, spoiled], axis=1)


def run_attend(device, cache, q, table, lengths, starts, scale, dtype, lists=None, sinks=None, most=None, **kw):
    """Through strided queries and a strided output, checked against the definition."""
    qt, qf = rounded(q, dtype)
    tokens, heads, d = q.shape
    wide = torch.full((tokens + 2, heads + 1, d), float("nan"), dtype=TYPES[dtype])
    wide[:tokens, :heads] = qt
    out = torch.full((tokens + 2, heads, d), 7.0, dtype=TYPES[dtype], device=device)
    wide = wide.to(device)
    most = most or max(1, int(np.diff(starts).max()))
    want, far = plain.attend(cache, qf, table, lengths.tolist(), starts.tolist(), scale, dtype, picked=lists, sinks=sinks, **kw)
    want, far = want[:starts[-1]], far[:starts[-1]]
    for form in (table, widened(table, cache, tokens, most, heads)) if lists is None else (table,):
        out[:tokens] = 7.0
        got = ops.paged_attend(to_device(cache, device), wide[:tokens, :heads], dev(form, device), dev(lengths, device), dev(starts, device), scale,
                               lists=None if lists is None else dev(lists, device), sinks=None if sinks is None else dev(sinks, device),
                               most=most, out=out[:tokens], **kw)
        x = got[:starts[-1]].double().cpu().numpy()
        near = np.abs(x - want) <= far
        if not near.all():
            at = np.argwhere(~near)
            worst = np.nanmax(np.abs(x - want) / np.maximum(far, 1e-30))
            pytest.fail(f"{len(at)} of {near.size} values too far off, up to {worst} of the distance; the first at {at[:4].tolist()}: {x[tuple(at[0])]}, not {want[tuple(at[0])]}")
        assert bool((out[starts[-1]:] == 7.0).all())  # rows of no request stay as they are
    return x, want


GEOMETRIES = [(4, 2, 64, 16), (32, 8, 128, 64), (16, 8, 256, 32), (7, 1, 128, 48), (14, 2, 64, 128), (6, 6, 256, 256), (24, 1, 64, 64), (40, 2, 128, 16)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,d,page", GEOMETRIES)
def test_decode_steps_at_lengths_around_pages_and_tiles(device, dtype, heads, kv_heads, d, page):
    g = np.random.default_rng(heads * d + page)
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300, 511, 1000]
    fresh = [1] * len(lengths)
    fresh[4] = fresh[9] = 0  # requests with nothing new
    cache, table, lengths, starts = serving(g, lengths, fresh, kv_heads, page, d)
    q = g.standard_normal((starts[-1], heads, d)) * 2
    run_attend(device, cache, q, table, lengths, starts, d ** -0.5, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window,softcap,with_sinks", [(0, 0.0, False), (1, 0.0, True), (37, 20.0, False), (100, 0.0, True), (5000, 50.0, True)])
def test_drafts_and_prompts_with_windows_softcaps_and_sinks(device, dtype, window, softcap, with_sinks):
    for heads, kv_heads, d, page in [(4, 2, 64, 16), (8, 2, 128, 64), (6, 1, 256, 32)]:
        g = np.random.default_rng(window + d)
        fresh = [3, 1, 40, 9, 0, 70, 2]
        cache, table, lengths, starts = serving(g, [500, 1, 40, 260, 64, 75, 2], fresh, kv_heads, page, d)
        q = g.standard_normal((starts[-1], heads, d)) * 3
        sinks = (g.standard_normal(heads) * 3).astype(np.float32) if with_sinks else None
        run_attend(device, cache, q, table, lengths, starts, d ** -0.5, dtype, window=window, softcap=softcap, sinks=sinks)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(4, 2, 64, 16), (8, 2, 128, 64), (4, 2, 256, 48), (1, 1, 128, 32), (24, 1, 64, 128)])
def test_prompts_of_odd_lengths(device, dtype, heads, kv_heads, d, page):
    g = np.random.default_rng(heads + d + page)
    fresh = [257, 1, 129, 33, 64]
    cache, table, lengths, starts = serving(g, [257, 300, 333, 33, 700], fresh, kv_heads, page, d)
    q = g.standard_normal((starts[-1], heads, d)) * 2
    for window in (0, 50):
        run_attend(device, cache, q, table, lengths, starts, d ** -0.5, dtype, window=window)


@pytest.mark.parametrize("longest", [200, 1600])
def test_prompts_beside_decoding_requests(device, longest):
    """Decoding requests that the prompts' form takes along, and more of them than it does."""
    g = np.random.default_rng(longest)
    fresh = [100, 0, 17] + [1] * 40 + [33]
    lengths = [400, 9, 100] + [longest - 7 * i % 160 for i in range(40)] + [33]
    cache, table, lengths, starts = serving(g, lengths, fresh, 2, 16, 64)
    run_attend(device, cache, g.standard_normal((starts[-1], 8, 64)), table, lengths, starts, 0.125, "f16")


@pytest.mark.parametrize("requests,kv_heads,d", [(70, 4, 128), (40, 2, 256), (130, 4, 64)])
def test_runs_of_a_workgroup_longer_than_a_round(device, requests, kv_heads, d):
    """Segments of unlike lengths, as many tiles as make a workgroup's run several rounds of its waves: whole segments and cut ones."""
    g = np.random.default_rng(requests)
    lengths = [int(n) for n in g.integers(700, 1100, requests)]
    lengths[3], lengths[-1] = 1, 2900
    cache, table, lengths, starts = serving(g, lengths, [1] * requests, kv_heads, 32, d)
    run_attend(device, cache, g.standard_normal((requests, 2 * kv_heads, d)), table, lengths, starts, d ** -0.5, "bf16")


def test_a_prompt_among_more_requests_than_the_list_takes_at_once(device):
    g = np.random.default_rng(1101)
    fresh = [1, 0, 2, 1, 1] * 230
    fresh[7], fresh[1100] = 90, 40
    lengths = [max(n, int(g.integers(0, 120))) for n in fresh]
    cache, table, lengths, starts = serving(g, lengths, fresh, 1, 16, 64)
    run_attend(device, cache, g.standard_normal((starts[-1], 4, 64)), table, lengths, starts, 0.125, "bf16")


@pytest.mark.parametrize("fresh", [0, 1, 5, 33, 100])
def test_one_request_of_fewer_tokens_than_rows(device, fresh):
    """The rows' count says what may come, the starts what does: a captured step answers both."""
    g = np.random.default_rng(fresh + 17)
    cache, table, lengths, starts = serving(g, [300], [fresh], 2, 16, 64)
    run_attend(device, cache, g.standard_normal((100, 8, 64)), table, lengths, starts, 0.125, "bf16", most=100)


def test_rows_that_see_nothing_are_zero(device):
    """More queries than a request has tokens (the first ones are before position 0), pages that are not in the cache."""
    g = np.random.default_rng(11)
    for fresh in ([5, 2, 1, 3], [5, 200, 1, 150]):
        cache, table, lengths, starts = serving(g, [2, 0, 64, 40], fresh, 2, 16, 64)
        table[2, :4] = [-1, 99999, -1, -1]
        q = g.standard_normal((starts[-1], 4, 64))
        for sinks in (None, g.standard_normal(4).astype(np.float32)):
            x, _ = run_attend(device, cache, q, table, lengths, starts, 0.125, "f32", sinks=sinks)
            assert np.all(x[:3] == 0) and np.all(x[starts[1]:starts[2]] == 0) and np.all(x[starts[2]:starts[3]] == 0) and np.any(x[3] != 0)


@pytest.mark.parametrize("fresh", [1, 60])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scales_of_any_size_and_spoiled_tokens(device, dtype, fresh):
    """V scales that differ by twelve orders of magnitude, pages of zero scale, K of zero scale; spoiled scales in a page that only later rows see."""
    g = np.random.default_rng(21)
    cache, table, lengths, starts = serving(g, [640, 200], [fresh, fresh], 2, 16, 128)
    cache["v_scale"][:] = np.where(np.isnan(cache["v_scale"]), np.nan, 10.0 ** g.uniform(-8, 4, cache["v_scale"].shape)).astype(np.float32)
    cache["v_scale"][table[0, 3]] = 0.0
    cache["k_scale"][table[0, 4]] = 0.0
    cache["v_scale"][table[1, :13]] = 0.0  # everything the second request sees
    q = g.standard_normal((starts[-1], 4, 128)) * 2
    x, _ = run_attend(device, cache, q, table, lengths, starts, 128 ** -0.5, dtype)
    assert np.all(x[starts[1]:] == 0)
    if fresh > 16:  # the last page's scales are not numbers: rows before it do not notice
        spoiled = {name: np.array(x) for name, x in cache.items()}
        for name in ("k_scale", "v_scale"):
            spoiled[name][table[0, 39]] = np.nan
        for form in (table, widened(table, cache, len(q), fresh, 4)):
            clean, got = [ops.paged_attend(to_device(c, device), rounded(q, dtype)[0].to(device), dev(form, device), dev(lengths, device),
                                           dev(starts, device), 0.1) for c in (cache, spoiled)]
            assert torch.equal(got[:44], clean[:44]) and bool(torch.isnan(got[44:60]).all()) and torch.equal(got[60:], clean[60:])


@pytest.mark.parametrize("fresh", [1, 40])
def test_a_query_that_is_no_number_spoils_its_own_row_only(device, fresh):
    g = np.random.default_rng(31)
    cache, table, lengths, starts = serving(g, [300, 90], [fresh, fresh], 2, 32, 64)
    c, n, s = to_device(cache, device), dev(lengths, device), dev(starts, device)
    values = torch.from_numpy(g.standard_normal((starts[-1], 8, 64)).astype(np.float32)).to(device)
    for form in (table, widened(table, cache, starts[-1], fresh, 8)):
        t, q = dev(form, device), values.clone()
        clean = ops.paged_attend(c, q, t, n, s, 0.125)
        q[0, 3, 9], q[-1, 5, 0] = float("nan"), float("inf")
        got = ops.paged_attend(c, q, t, n, s, 0.125)
        spoiled = torch.zeros_like(got, dtype=torch.bool)
        spoiled[0, 3], spoiled[-1, 5] = True, True
        assert bool(torch.isnan(got[spoiled]).all()) and torch.equal(got[~spoiled], clean[~spoiled])
        q[0, 3], q[-1, 5] = 0.0, 0.0  # zeros: the plain mean of what is seen
        got = ops.paged_attend(c, q, t, n, s, 0.125)
        k, v = plain.values(cache, table[0, :10])
        p = 300 - fresh + 1
        mean = np.swapaxes(v, 0, 1).reshape(2, -1, 64)[:, :p].mean(1)
        assert np.allclose(got[0, 3].cpu().numpy(), mean[0], rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_many_requests_and_a_long_one(device, dtype):
    g = np.random.default_rng(41)
    lengths = [4000] + [int(x) for x in g.integers(1, 60, 149)]
    fresh = [1] + [int(x) for x in g.integers(0, 4, 149)]
    fresh = [min(f, n) for f, n in zip(fresh, lengths)]
    cache, table, lengths, starts = serving(g, lengths, fresh, 1, 16, 128)
    q = g.standard_normal((starts[-1], 5, 128))
    run_attend(device, cache, q, table, lengths, starts, 0.088, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(4, 2, 64, 16), (32, 8, 128, 64), (20, 1, 256, 48)])
def test_lists_leave_their_pages_only(device, dtype, heads, kv_heads, d, page):
    g = np.random.default_rng(51 + page)
    cache, table, lengths, starts = serving(g, [900, 33, 500, 1], [3, 2, 1, 1], kv_heads, page, d)
    q = g.standard_normal((starts[-1], heads, d)) * 2
    keep = 7
    lists = np.full((starts[-1], kv_heads, keep), -1, dtype=np.int32)
    for r in range(4):
        for t in range(starts[r], starts[r + 1]):
            n = plain.ceil(int(lengths[r]), page)
            for h in range(kv_heads):
                some = np.sort(g.permutation(n)[:g.integers(0, keep + 1)])
                lists[t, h, :len(some)] = some
    lists[0, 0] = -1  # nothing at all
    lists[1, 0] = [table.shape[1], 5000000, -9, 0, -1, 1, 1 << 30]  # places past the table
    for window in (0, 100):
        run_attend(device, cache, q, table, lengths, starts, d ** -0.5, dtype, lists=lists, window=window)


def test_pages_past_four_gigabytes(device):
    """Codes whose byte offset passes 32 bits: a decode step, a prompt, the store and the selection at the end of the cache."""
    pages, kv_heads, page, d = 70000, 4, 128, 128
    big = ops.paged_cache(pages, kv_heads, page, d, device)
    assert big["k"].numel() > 1 << 32
    g = np.random.default_rng(61)
    small = random_cache(g, 8, kv_heads, page, d)
    at = np.array([69999, 66000, 3, 69000, 68123, 67777, 69998, 65999])
    for name in small:
        big[name][dev(at, device)] = dev(small[name], device)
    table = at[None].astype(np.int32)
    x = g.standard_normal((2, 10, kv_heads, d)).astype(np.float32)
    work = np.array([[69998, 0, 20, 10]], dtype=np.int32)
    ops.paged_store(big, dev(x[0], device), dev(x[1], device), dev(work, device))
    plain.store(small, x[0], x[1], [[6, 0, 20, 10]])
    same(big["k"][69998], small["k"][6], "k")
    same(big["v"][69998], small["v"][6], "v")
    back = ops.paged_read(big, dev(table[0], device))
    same(back[1], np.swapaxes(small["v"], 2, 3).astype(np.float32) * small["v_scale"][..., None, None], "read")
    for fresh in (1, 70):
        lengths, starts = np.array([1000], dtype=np.int32), np.array([0, fresh], dtype=np.int32)
        q = g.standard_normal((fresh, 8, d)).astype(np.float32)
        here = np.arange(8, dtype=np.int32)[None]
        want, far = plain.attend(small, q, here, [1000], [0, fresh], 0.1, "f32")
        for form in (table, widened(table, small, fresh, fresh, 8)):
            got = ops.paged_attend(big, dev(q, device), dev(form, device), dev(lengths, device), dev(starts, device), 0.1).double().cpu().numpy()
            assert np.all(np.abs(got - want) <= far)
        got = ops.paged_select(big, dev(q, device), dev(table, device), dev(lengths, device), dev(starts, device), 4)
        same(got, plain.lists(small, q, here, [1000], [0, fresh], 4), "lists")


# ---------------------------------------------------------------- the selection


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(4, 2, 64, 16), (32, 8, 128, 64), (16, 8, 256, 32), (7, 1, 128, 16), (40, 2, 64, 16), (14, 2, 64, 48)])
def test_selection_is_its_definition(device, dtype, heads, kv_heads, d, page):
    g = np.random.default_rng(heads + d + page)
    fresh = [1, 3, 0, 20, 2, 1]
    cache, table, lengths, starts = serving(g, [page * 70 + 3, 40, 64, page * 21, 2, 1], fresh, kv_heads, page, d)
    qt, q = rounded(g.standard_normal((starts[-1] + 2, heads, d)), dtype)
    for keep, first, recent in [(1, 0, 1), (2, 1, 1), (9, 0, 0), (20, 3, 4), (200, 1, 1)]:
        got = ops.paged_select(to_device(cache, device), qt.to(device), dev(table, device), dev(lengths, device), dev(starts, device), keep,
                               first=first, recent=recent, most=20)
        want = plain.lists(cache, q, table, lengths, starts, keep, first, recent)
        same(got, want, f"keep {keep}")


def test_selection_ties_zeros_and_queries_that_are_no_numbers(device):
    g = np.random.default_rng(71)
    cache, table, lengths, starts = serving(g, [16 * 600], [5], 1, 16, 64)
    cache["low"][:], cache["high"][:] = -3, 5  # every page the same bound but for its scale
    cache["k_scale"][:] = 0.25
    cache["k_scale"][table[0, 100:130]] = 0.5
    q = g.standard_normal((5, 3, 64)).astype(np.float32)
    q[1] = 0.0
    q[2, 0, 0], q[2, 1, 5], q[2, 2, 9] = np.nan, np.inf, -np.inf  # no score at all
    q[3, 1, 7] = np.nan  # the other heads' scores
    q[4] *= 1e-38
    for keep in (4, 40, 300):
        got = ops.paged_select(to_device(cache, device), dev(q, device), dev(table, device), dev(lengths, device), dev(starts, device), keep)
        same(got, plain.lists(cache, q, table, lengths, starts, keep), f"keep {keep}")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(8, 1, 64, 16), (16, 4, 128, 16), (2, 2, 256, 48), (32, 2, 128, 32)])
def test_selection_of_many_tokens(device, dtype, heads, kv_heads, d, page):
    """As many rows as one launch takes (above), with requests of no fresh tokens, of one page, and rows of no request."""
    g = np.random.default_rng(heads + d + page + 1)
    fresh = ([1, 0, 7, 1, 16, 2, 3, 1] * 24)[:190]
    fresh[40] = 33
    held = [max(n, int(g.integers(0, 60 * page))) for n in fresh]
    held[1], held[9] = 0, 0
    held[40], held[41] = page * 80, page * 300 - 1
    cache, table, lengths, starts = serving(g, held, fresh, kv_heads, page, d)
    tokens = int(starts[-1])
    qt, q = rounded(g.standard_normal((tokens + 3, heads, d)), dtype)
    cache["k_scale"][table[41, 100:130]] = 0.5
    cache["low"][table[41, 100:130]], cache["high"][table[41, 100:130]] = -3, 5
    q[4, 0, 3] = qt[4, 0, 3] = np.nan
    q[6], qt[6] = 0.0, 0.0
    for keep, first, recent in [(1, 0, 1), (9, 0, 0), (20, 3, 4), (6, 2, 4), (70, 1, 1)]:
        got = ops.paged_select(to_device(cache, device), qt.to(device), dev(table, device), dev(lengths, device), dev(starts, device), keep,
                               first=first, recent=recent)
        same(got, plain.lists(cache, q, table, lengths, starts, keep, first, recent), f"keep {keep}")


def test_selection_of_more_pages_than_a_workgroup_keeps(device):
    g = np.random.default_rng(72)
    pages = 20011
    cache = {k: v for k, v in random_cache(g, pages, 1, 16, 64).items()}
    table = g.permutation(pages).astype(np.int32)[None]
    lengths, starts = np.array([pages * 16 - 5], dtype=np.int32), np.array([0, 2], dtype=np.int32)
    q = g.standard_normal((2, 4, 64)).astype(np.float32)
    cache["low"], cache["high"] = g.integers(-127, 0, cache["low"].shape).astype(np.int8), g.integers(0, 128, cache["low"].shape).astype(np.int8)
    got = ops.paged_select(to_device(cache, device), dev(q, device), dev(table, device), dev(lengths, device), dev(starts, device), 1000)
    same(got, plain.lists(cache, q, table, lengths, starts, 1000), "lists")


# ---------------------------------------------------------------- together


def test_a_server_of_the_operators(device):
    """Steps as a program runs them: plan, store, attend (dense, and over selected pages that are all of them), on a stream of its own; what the
    cache gives back is near what went in."""
    g = np.random.default_rng(81)
    kv_heads, heads, page, d, requests = 2, 8, 16, 64, 6
    cache = ops.paged_cache(40, kv_heads, page, d, device)
    table = torch.full((requests, 12), -1, dtype=torch.int32, device=device)
    ring = torch.arange(40, dtype=torch.int32, device=device)
    counters = torch.tensor([0, 40, 0], dtype=torch.int32, device=device)
    keys = [np.zeros((0, kv_heads, d), np.float32)] * requests
    vals = [np.zeros((0, kv_heads, d), np.float32)] * requests
    held = np.zeros(requests, dtype=np.int32)
    steps = [[30, 1, 0, 17, 5, 0], [1, 1, 50, 1, 1, 0], [1, -1, 1, 1, 1, 16], [1, 1, 1, -1, 3, 1], [2, 20, 1, 33, 1, 1]]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for step in steps:
            step = np.array(step)
            after = np.where(step < 0, 0, held + step).astype(np.int32)
            rows = int(np.maximum(after - held, 0).sum())
            k, v, q = (g.standard_normal((rows, n, d)).astype(np.float32) for n in (kv_heads, kv_heads, heads))
            plan = ops.paged_plan(dev(held, device), dev(after, device), table, ring, counters, page, rows)
            counters = plan["counters"]
            ops.paged_store(cache, dev(k, device), dev(v, device), plan["work"])
            got = ops.paged_attend(cache, dev(q, device), table, plan["lengths"], plan["starts"], 0.125)
            lists = ops.paged_select(cache, dev(q, device), table, plan["lengths"], plan["starts"], 12)
            over = ops.paged_attend(cache, dev(q, device), table, plan["lengths"], plan["starts"], 0.125, lists=lists)
            assert torch.allclose(got, over, rtol=1e-4, atol=1e-5)
            at = 0
            for r in range(requests):
                n = max(int(after[r] - held[r]), 0)
                keep = int(min(held[r], after[r]))
                keys[r], vals[r] = (np.concatenate([x[r][:keep], y[at:at + n]]) for x, y in ((keys, k), (vals, v)))
                for t in range(n):
                    p = int(after[r]) - n + t
                    for h in range(heads):
                        s = keys[r][:p + 1, h // 4] @ q[at + t, h] * 0.125
                        w = np.exp(s - s.max())
                        want = w @ vals[r][:p + 1, h // 4] / w.sum()
                        assert np.abs(got[at + t, h].cpu().numpy() - want).max() <= 0.1  # (8-bit codes of values near 4)
                at += n
            held = after
    stream.synchronize()
    assert counters.cpu().tolist()[2] == 0


@pytest.mark.parametrize("keep", [0, 3])
def test_the_example_server(device, keep):
    """examples/paged_server.py: two layers on one plan, requests that come, answer and end, against the definition over each cache."""
    spec = importlib.util.spec_from_file_location("paged_server", os.path.join(os.path.dirname(__file__), "..", "examples", "paged_server.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    g = np.random.default_rng(97)
    server = module.PagedServer(3, 24, 8, layers=2, heads=8, kv_heads=2, head_dim=64, page=16, keep=keep, device=device)
    for after in ([100, 0, 33], [101, 1, 34], [102, 40, 0], [103, 41, 1], [0, 42, 2]):
        before = server.lengths.cpu().numpy()
        fresh = np.maximum(np.array(after) - before, 0)
        rows = [[g.standard_normal((fresh.sum(), h, 64)).astype(np.float32) for h in (8, 2, 2)] for _ in range(2)]
        x, plan = server.step(dev(np.array(after, dtype=np.int32), device), int(fresh.sum()), int(fresh.max()),
                              lambda layer, x: [dev(v, device) for v in rows[layer]])
        assert plan["counters"][2].item() == 0 and plan["lengths"].tolist() == after
        cache = {name: v.cpu().numpy() for name, v in server.caches[1].items()}
        table, starts = server.table.cpu().numpy(), plan["starts"].tolist()
        lists = plain.lists(cache, rows[1][0], table, after, starts, keep) if keep and fresh.max() == 1 else None
        want, far = plain.attend(cache, rows[1][0], table, after, starts, 0.125, "f32", picked=lists)
        assert np.all(np.abs(x.double().cpu().numpy() - want) <= far)


def test_captured_launches_replay_at_other_lengths(device):
    g = np.random.default_rng(91)
    cache, table, lengths, starts = serving(g, [700, 300, 90], [1, 1, 1], 2, 16, 128)
    c, t = to_device(cache, device), dev(table, device)
    q = dev(g.standard_normal((3, 8, 128)).astype(np.float32), device)
    n, s = dev(lengths, device), dev(starts, device)
    lib = _lib.load()
    out, lists, over = torch.empty_like(q), torch.empty((3, 2, 6), dtype=torch.int32, device=device), torch.empty_like(q)
    scratch = torch.empty(64 << 20, dtype=torch.uint8, device=device)
    scores = torch.empty(16 << 20, dtype=torch.uint8, device=device)

    def work():
        ops.paged_attend(c, q, t, n, s, 0.088, most=1, out=out, scratch=scratch)
        ops.paged_select(c, q, t, n, s, 6, most=1, out=lists, scratch=scores)
        ops.paged_attend(c, q, t, n, s, 0.088, lists=lists, most=1, out=over, scratch=scratch)

    assert lib is not None
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for step, now in enumerate([[700, 300, 90], [17, 299, 1], [650, 64, 65], [1, 1, 90]]):
        n.copy_(torch.tensor(now, dtype=torch.int32))
        q.copy_(dev(g.standard_normal((3, 8, 128)).astype(np.float32), device))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in (out, lists, over)]
        work()
        torch.cuda.synchronize()
        for a, b in zip(replayed, (out, lists, over)):
            assert torch.equal(a, b), f"replay {step}"
        want, far = plain.attend(cache, q.cpu().numpy(), table, now, starts.tolist(), 0.088, "f32")
        assert np.all(np.abs(out.double().cpu().numpy() - want) <= far)


def test_captured_prompts_and_selections_replay_at_other_lengths(device):
    """The launches of a step of at most 300 tokens, the prompts' form and a selection in one launch among them, with other tokens a request."""
    g = np.random.default_rng(93)
    cache, table, lengths, starts = serving(g, [900, 500, 400], [200, 60, 40], 4, 16, 64)
    table = widened(table, cache, 300, 300, 16)
    c, t = to_device(cache, device), dev(table[:, :80], device)
    wide, n, s = dev(table, device), dev(lengths, device), dev(starts, device)
    q = dev(g.standard_normal((300, 16, 64)).astype(np.float32), device)
    out, lists = torch.zeros_like(q), torch.zeros((300, 4, 6), dtype=torch.int32, device=device)
    scratch, scores = torch.empty(256 << 20, dtype=torch.uint8, device=device), torch.empty(16 << 20, dtype=torch.uint8, device=device)

    def work():
        ops.paged_attend(c, q, wide, n, s, 0.125, most=300, out=out, scratch=scratch)
        ops.paged_select(c, q, t, n, s, 6, most=300, out=lists, scratch=scores)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for step, (now, fresh) in enumerate([([900, 500, 400], [200, 60, 40]), ([17, 299, 1], [17, 250, 1]), ([650, 64, 400], [0, 1, 299]), ([900, 500, 400], [1, 1, 1])]):
        n.copy_(torch.tensor(now, dtype=torch.int32))
        begins = [0, fresh[0], fresh[0] + fresh[1], sum(fresh)]
        s.copy_(torch.tensor(begins, dtype=torch.int32))
        q.copy_(dev(g.standard_normal((300, 16, 64)).astype(np.float32), device))
        scratch.random_(0, 256)  # what a call before left there is no matter
        out.zero_(), lists.zero_()
        graph.replay()
        torch.cuda.synchronize()
        end = begins[3]
        want, far = plain.attend(cache, q.cpu().numpy(), table, now, begins, 0.125, "f32")
        assert np.all(np.abs(out[:end].double().cpu().numpy() - want[:end]) <= far[:end]), f"replay {step}"
        assert bool((out[end:] == 0).all())
        same(lists, plain.lists(cache, q.cpu().numpy(), table, now, begins, 6), f"replay {step}")


def test_seeded_inputs_are_what_synth_gives(device):
    """The benchmark's own activations through the cache: BF16 values that many codes hold."""
    x = synth.bf16_to_f32(synth.bf16_bits(synth.activations(64, 256, 3))).reshape(64, 2, 128)
    cache = ops.paged_cache(4, 2, 16, 128, device)
    host = {k: v.cpu().numpy() for k, v in cache.items()}
    work = [[3, 0, 0, 16], [1, 16, 0, 16], [0, 32, 0, 16], [2, 48, 0, 16]]
    xd = dev(x, device).to(torch.bfloat16)
    ops.paged_store(cache, xd, xd, dev(np.array(work, dtype=np.int32), device))
    plain.store(host, x, x, work)
    for name in host:
        same(cache[name], host[name], name)
