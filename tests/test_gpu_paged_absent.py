"""llmp_hip_paged_select over table entries that are no pages of the cache: they have no score, are never chosen, and the attention
over what is chosen is the one over all that is there where the list has room for it."""
import numpy as np
import pytest
import torch

import paged_plain as plain
from llmp_amd import ops
from test_gpu_paged import dev, random_cache, rounded, same, serving, to_device

pytestmark = pytest.mark.gpu

ABSENT = np.array([-1, -7, 1 << 30, -(1 << 31), 2147483647], dtype=np.int32)


def lists(cache, q, table, lengths, starts, keep, first, recent):
    """The definition, a row and a KV head at a time, over the pages that are there."""
    pages, kv_heads, page, d = cache["k"].shape
    group = q.shape[1] // kv_heads
    one = np.float32
    out = np.full((len(q), kv_heads, keep), -1, dtype=np.int32)
    for r in range(len(lengths)):
        for t in range(starts[r], starts[r + 1]):
            seen = int(lengths[r] - starts[r + 1] + t) + 1
            n = plain.ceil(max(seen, 0), page)
            places = [j for j in range(n) if 0 <= table[r, j] < pages]
            at = table[r, places]
            for h in range(kv_heads):
                score = np.full(len(places), -np.inf, dtype=np.float32)
                for x in q[t, h * group:(h + 1) * group].astype(np.float32):
                    unit = np.abs(x).max() * (one(1) / one(127))
                    c = np.clip(np.rint(x / unit), -127, 127).astype(np.float64)
                    bound = np.where(c > 0, c * cache["high"][at, h], c * cache["low"][at, h]).sum(1).astype(np.float32)
                    score = np.maximum(score, (bound * unit) * cache["k_scale"][at, h])
                rank = sorted(range(len(places)), key=lambda i: (not (places[i] < first or places[i] >= n - recent), -score[i], places[i]))
                chosen = sorted(places[i] for i in rank[:keep])
                out[t, h, :len(chosen)] = chosen
    return out


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,d,page,copies", [(4, 2, 64, 16, 1), (32, 8, 128, 32, 4), (7, 1, 256, 48, 1), (16, 8, 64, 16, 5)])
def test_pages_that_are_not_there_are_not_chosen(device, dtype, heads, kv_heads, d, page, copies):
    """Absent pages among the scored, the first and the recent ones, requests of which few pages are left, or none. A page 0 whose bound is
    above all others' would be chosen for any of them. By `copies` of the requests the two launches or the one."""
    g = np.random.default_rng(heads + d + page)
    fresh = [1, 5, 3, 2, 1, 7] * copies
    held = [page * 70 + 3, page * 23, page * 12 + 1, 40, page * 9, page * 33 - 2] * copies
    cache, table, lengths, starts = serving(g, held, fresh, kv_heads, page, d)
    cache["low"][0], cache["high"][0], cache["k_scale"][0] = -127, 127, 5.0
    table[table == 0] = 1
    for r, n in enumerate(held):
        n = plain.ceil(n, page)
        gone = [g.random(n) < 0.2, np.arange(n) % 2 == 0, np.arange(n) != 3, np.ones(n, bool), np.arange(n) == n - 1, np.arange(n) < 4][r % 6]
        table[r, :n] = np.where(gone, g.choice(ABSENT, n), table[r, :n])
    table[1, 2] = len(cache["k"])  # the first number past the cache
    qt, q = rounded(g.standard_normal((starts[-1] + 2, heads, d)), dtype)
    c, t, n, s, x = to_device(cache, device), dev(table, device), dev(lengths, device), dev(starts, device), qt.to(device)
    for keep, first, recent in [(1, 0, 1), (4, 1, 1), (9, 0, 0), (20, 9, 11), (30, 3, 4), (table.shape[1], 1, 1), (100, 0, 2)]:
        same(ops.paged_select(c, x, t, n, s, keep, first=first, recent=recent), lists(cache, q, table, lengths, starts, keep, first, recent), f"keep {keep}")


def test_more_pages_than_a_workgroup_keeps_and_some_of_them_gone(device):
    g = np.random.default_rng(3)
    pages = 9001
    cache = random_cache(g, pages, 1, 16, 64)
    table = g.permutation(pages).astype(np.int32)[None]
    table[0, g.random(pages) < 0.4] = -1
    lengths, starts = np.array([pages * 16 - 5], dtype=np.int32), np.array([0, 2], dtype=np.int32)
    q = g.standard_normal((2, 4, 64)).astype(np.float32)
    there = int((table >= 0).sum())
    for keep in (700, 4096):
        got = ops.paged_select(to_device(cache, device), dev(q, device), dev(table, device), dev(lengths, device), dev(starts, device), keep)
        same(got, lists(cache, q, table, lengths, starts, keep, 1, 1), f"keep {keep} of {there}")


@pytest.mark.parametrize("kv_heads", [2, 64])
def test_a_list_with_room_for_all_that_is_there(device, kv_heads):
    g = np.random.default_rng(kv_heads)
    cache, table, lengths, starts = serving(g, [16 * 40, 16 * 33 + 5], [2, 3], kv_heads, 16, 64)
    table[:, 5:25] = -1
    q = torch.from_numpy(g.standard_normal((5, 2 * kv_heads, 64)).astype(np.float32)).to(device)
    where = to_device(cache, device), q, dev(table, device), dev(lengths, device), dev(starts, device)
    for keep in (20, 64):
        picked = ops.paged_select(*where, keep)
        assert picked[0, 0].tolist() == [0, 1, 2, 3, 4] + list(range(25, 40)) + [-1] * (keep - 20)
        assert torch.allclose(ops.paged_attend(*where, 0.125, lists=picked), ops.paged_attend(*where, 0.125), rtol=1e-4, atol=1e-5)
