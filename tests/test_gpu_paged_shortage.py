"""Steps of the paged cache whose pages run out, and lengths that end before a request's new tokens (llmp_hip_paged_attend and
_select with `before`): a token past what is held keeps its position and sees all that is held."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import paged_plain as plain
from llmp_amd import ops
from test_gpu_paged import dev, random_cache, rounded, same, to_device, widened

pytestmark = pytest.mark.gpu


def rows_of(lengths, before, starts):
    """(row, request, position, end of what it sees) of every new token."""
    for r in range(len(lengths)):
        for t in range(starts[r + 1] - starts[r]):
            p = int(before[r]) + t
            yield starts[r] + t, r, p, min(p + 1, int(lengths[r]))


def attend(cache, q, table, lengths, before, starts, scale, dtype, window=0, picked=None, **kw):
    """paged_plain.attend a row at a time: a token at p that sees up to `end` has what one at end - 1 has, its window shorter by
    what lies between."""
    out, far = np.zeros(q.shape), np.zeros(q.shape)
    for row, r, p, end in rows_of(lengths, before, starts):
        left = window - (p + 1 - end) if window else 0
        if end > 0 and (not window or left > 0):
            x, y = plain.attend(cache, q[row:row + 1], table[r:r + 1], [end], [0, 1], scale, dtype, window=left,
                                picked=None if picked is None else picked[row:row + 1], **kw)
            out[row], far[row] = x[0], y[0]
    return out, far


def lists(cache, q, table, lengths, before, starts, keep, **kw):
    out = np.full((len(q), cache["k"].shape[1], keep), -1, dtype=np.int32)
    for row, r, p, end in rows_of(lengths, before, starts):
        if end > 0:
            out[row] = plain.lists(cache, q[row:row + 1], table[r:r + 1], [end], [0, 1], keep, **kw)[0]
    return out


def near(got, want, far, name):
    wrong = ~(np.abs(got.double().cpu().numpy() - want) <= far)
    assert not wrong.any(), f"{name}: {int(wrong.sum())} of {wrong.size} values too far off, rows {sorted(set(np.argwhere(wrong)[:, 0].tolist()))[:9]}"


def check(device, cache, q, table, lengths, before, starts, dtype, keep=3):
    """The attention in both forms, with and without a window, the selection, and the attention over what it selects."""
    qt, q = rounded(q, dtype)
    c, qt, n, b, s = to_device(cache, device), qt.to(device), dev(lengths, device), dev(before, device), dev(starts, device)
    tokens, heads, d = q.shape
    most = int(np.diff(starts).max())
    for window in (0, 30):
        want, far = attend(cache, q, table, lengths, before, starts, d ** -0.5, dtype, window=window)
        for form in (table, widened(table, cache, tokens, most, heads)):
            got = ops.paged_attend(c, qt, dev(form, device), n, s, d ** -0.5, before=b, window=window, most=most)
            near(got, want, far, f"window {window}, {form.shape[1]} pages a row")
    want = lists(cache, q, table, lengths, before, starts, keep)
    picked = ops.paged_select(c, qt, dev(table, device), n, s, keep, before=b, most=most)
    same(picked, want, "lists")
    got = ops.paged_attend(c, qt, dev(table, device), n, s, d ** -0.5, before=b, lists=picked, most=most)
    near(got, *attend(cache, q, table, lengths, before, starts, d ** -0.5, dtype, picked=want), "over the lists")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kv_heads,page,d,free", [(1, 16, 64, 9), (8, 16, 64, 5), (2, 32, 128, 3), (2, 16, 256, 0)])
def test_a_step_whose_pages_run_out(device, dtype, kv_heads, page, d, free):
    """A decode step on a page's edge, drafts, prompts (the one that finds some pages, and those after it none, one of them
    with nothing held), one token that needs no page: plan, store and what reads it."""
    g = np.random.default_rng(page + d + free)
    before = np.array([page * 3, page * 5 - 3, 10, page * 2 + 1, 0, page - 2, 7], dtype=np.int32)
    fresh = np.array([1, 6, 100, 40, 20, 1, 0], dtype=np.int32)
    have = [plain.ceil(int(n), page) for n in before]
    pages, width = sum(have) + free + 1, plain.ceil(int((before + fresh).max()), page)
    order = g.permutation(pages).astype(np.int32)
    table, at = np.full((7, width), -1, dtype=np.int32), 0
    for r, n in enumerate(have):
        table[r, :n], at = order[at:at + n], at + n
    ring = np.concatenate([order[at:at + free], np.zeros(max(0, 1 - free), dtype=np.int32)])
    cache = random_cache(g, pages, kv_heads, page, d)
    starts = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
    c, t = to_device(cache, device), dev(table, device)
    plan = ops.paged_plan(dev(before, device), dev(before + fresh, device), t, dev(ring, device), dev(np.array([0, free, 0], np.int32), device), page,
                          int(starts[-1]))
    k, v = (rounded(g.standard_normal((starts[-1], kv_heads, d)), dtype) for _ in range(2))
    ops.paged_store(c, k[0].to(device), v[0].to(device), plan["work"])
    lengths = plan["lengths"].cpu().numpy()
    assert plan["counters"][2].item() == int((before + fresh - lengths).sum()) > 0 and plan["starts"].tolist() == starts.tolist()
    # (Every token of a page has a slot there and the others none: the positions are the plan's.)
    positions = plan["positions"].tolist()
    assert positions == [p for _, _, p, _ in rows_of(lengths, before, starts)]
    stored = {name: x.cpu().numpy() for name, x in c.items()}
    check(device, stored, g.standard_normal((starts[-1], 4 * kv_heads, d)), t.cpu().numpy(), lengths, before, starts, dtype)


@pytest.mark.parametrize("kv_heads", [1, 8])
def test_lengths_that_end_inside_a_page(device, kv_heads):
    """Whatever the lengths are: less than before, inside a page, none; and as long as before and the new tokens together, where
    `before` says what its absence does."""
    g = np.random.default_rng(kv_heads)
    before, fresh = np.array([40, 100, 0, 300, 5, 90], np.int32), np.array([30, 3, 25, 1, 90, 20], np.int32)
    lengths = np.array([53, 70, 0, 301, 6, 110], np.int32)
    cache = random_cache(g, 80, kv_heads, 16, 64)
    table = g.permutation(80)[:66].astype(np.int32).reshape(3, 22).repeat(2, 0)
    starts = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
    q = g.standard_normal((starts[-1], 4 * kv_heads, 64))
    check(device, cache, q, table, lengths, before, starts, "f32", keep=4)
    whole = before + fresh
    c, qt, t, s = to_device(cache, device), rounded(q, "bf16")[0].to(device), dev(table, device), dev(starts, device)
    for form in (t, dev(widened(table, cache, len(q), 90, 4 * kv_heads), device)):
        a, b = (ops.paged_attend(c, qt, form, dev(whole, device), s, 0.125, before=x) for x in (None, dev(before, device)))
        assert torch.equal(a, b)
    a, b = (ops.paged_select(c, qt, t, dev(whole, device), s, 4, before=x) for x in (None, dev(before, device)))
    assert torch.equal(a, b)


def test_the_example_server_whose_pages_run_out(device):
    spec = importlib.util.spec_from_file_location("paged_server", os.path.join(os.path.dirname(__file__), "..", "examples", "paged_server.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    g = np.random.default_rng(99)
    server = module.PagedServer(2, 5, 8, layers=1, heads=8, kv_heads=2, head_dim=64, page=16, device=device)
    missing = 0
    for grown in ([30, 0], [1, 20], [1, 20], [1, 1]):
        before = server.lengths.cpu().numpy()
        fresh = np.array(grown)
        rows = [g.standard_normal((fresh.sum(), h, 64)).astype(np.float32) for h in (8, 2, 2)]
        x, plan = server.step(dev((before + fresh).astype(np.int32), device), int(fresh.sum()), int(fresh.max()), lambda layer, x: [dev(v, device) for v in rows])
        missing += plan["counters"][2].item()
        cache = {name: v.cpu().numpy() for name, v in server.caches[0].items()}
        near(x, *attend(cache, rows[0], server.table.cpu().numpy(), plan["lengths"].tolist(), before, plan["starts"].tolist(), 0.125, "f32"), str(grown))
    assert missing > 0


def test_before_replays_with_the_launch(device):
    """A captured step of drafted tokens answers whatever before and lengths it finds."""
    g = np.random.default_rng(7)
    cache = random_cache(g, 40, 2, 16, 64)
    table = g.permutation(40)[:36].astype(np.int32).reshape(3, 12)
    starts = np.array([0, 4, 8, 12], np.int32)
    q = g.standard_normal((12, 8, 64)).astype(np.float32)
    c, t, s, x = to_device(cache, device), dev(table, device), dev(starts, device), dev(q, device)
    n, b = (torch.zeros(3, dtype=torch.int32, device=device) for _ in range(2))
    out, scratch = torch.zeros_like(x), torch.empty(64 << 20, dtype=torch.uint8, device=device)

    def work():
        ops.paged_attend(c, x, t, n, s, 0.125, before=b, most=4, out=out, scratch=scratch)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for before, lengths in (([30, 62, 0], [34, 64, 4]), ([31, 64, 0], [32, 64, 0]), ([100, 14, 3], [104, 16, 7])):
        b.copy_(torch.tensor(before, dtype=torch.int32))
        n.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        near(out, *attend(cache, q, table, lengths, before, starts, 0.125, "f32"), str(before))
        replayed = out.clone()
        work()
        torch.cuda.synchronize()
        assert torch.equal(out, replayed)


@pytest.mark.parametrize("window", [2147483647, 2147483646, 1 << 30, (1 << 30) - 1])
def test_a_window_past_every_position_hides_nothing(device, window):
    """Requests of fewer tokens than rows: their first positions lie before 0."""
    g = np.random.default_rng(5)
    cache = random_cache(g, 20, 2, 16, 64)
    table = g.permutation(20)[:12].astype(np.int32).reshape(2, 6)
    lengths, starts = np.array([40, 70], np.int32), np.array([0, 60, 135], np.int32)
    q = g.standard_normal((135, 8, 64)).astype(np.float32)
    c, x, n, s = to_device(cache, device), dev(q, device), dev(lengths, device), dev(starts, device)
    want, far = plain.attend(cache, q, table, lengths.tolist(), starts.tolist(), 0.125, "f32")
    for form in (table, widened(table, cache, 135, 75, 8)):
        got = ops.paged_attend(c, x, dev(form, device), n, s, 0.125, window=window)
        near(got, want, far, f"{form.shape[1]} pages a row")
        assert torch.equal(got, ops.paged_attend(c, x, dev(form, device), n, s, 0.125))


def test_one_token_of_a_row_of_odd_length(device):
    """A step of one token whose q, k and v are pieces of a row that no 16 bytes divide: its stride is not used."""
    g = np.random.default_rng(17)
    cache = random_cache(g, 4, 2, 16, 64)
    host, c = {name: x.copy() for name, x in cache.items()}, to_device(cache, device)
    rows = torch.from_numpy(g.standard_normal((3, 12 * 64 + 3)).astype(np.float32)).to(device)
    q, k, v = (rows[:, a * 64:b * 64].view(3, b - a, 64)[:1] for a, b in ((0, 8), (8, 10), (10, 12)))
    assert q.stride(0) % 4 != 0
    table, work = np.array([[2, 1]], np.int32), np.array([[1, 0, 3, 1]], np.int32)
    ops.paged_store(c, k, v, dev(work, device))
    plain.store(host, k.cpu().numpy(), v.cpu().numpy(), work.tolist())
    for name in host:
        same(c[name], host[name], name)
    where = dev(table, device), dev(np.array([20], np.int32), device), dev(np.array([0, 1], np.int32), device)
    near(ops.paged_attend(c, q, *where, 0.125), *plain.attend(host, q.cpu().numpy(), table, [20], [0, 1], 0.125, "f32"), "out")
    same(ops.paged_select(c, q, *where, 1, first=0), plain.lists(host, q.cpu().numpy(), table, [20], [0, 1], 1, first=0), "lists")
