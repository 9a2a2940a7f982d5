"""llmp_hip_paged_attend where its kernels take another way: scales below zero, and tables so wide that a unit of the work's line is several tiles."""
import numpy as np
import pytest
import torch

import paged_plain as plain
from llmp_amd import ops
from test_gpu_paged import dev, rounded, serving, to_device, widened

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("heads,kv_heads,d,page", [(8, 2, 64, 16), (8, 2, 128, 64), (4, 2, 256, 32)])
def test_a_scale_below_zero_is_the_query_turned(device, dtype, softcap, heads, kv_heads, d, page):
    g = np.random.default_rng(d + page)
    fresh = [70, 1, 0, 5, 40]
    cache, table, lengths, starts = serving(g, [300, 500, 3, 64, 41], fresh, kv_heads, page, d)
    qt, q = rounded(g.standard_normal((starts[-1], heads, d)) * 2, dtype)
    want, far = plain.attend(cache, -q, table, lengths.tolist(), starts.tolist(), d ** -0.5, dtype, softcap=softcap)
    c, x, n, s = to_device(cache, device), qt.to(device), dev(lengths, device), dev(starts, device)
    for form in (table, widened(table, cache, len(q), 70, heads)):
        got = ops.paged_attend(c, x, dev(form, device), n, s, -d ** -0.5, softcap=softcap)
        assert np.all(np.abs(got.double().cpu().numpy() - want) <= far)
    lists = dev(np.tile(np.array([0, 2, 3, -1], np.int32), (starts[-1], kv_heads, 1)), device)
    want, far = plain.attend(cache, -q, table, lengths.tolist(), starts.tolist(), d ** -0.5, dtype, softcap=softcap, picked=lists.cpu().numpy())
    got = ops.paged_attend(c, x, dev(table, device), n, s, -d ** -0.5, softcap=softcap, lists=lists)
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= far)


@pytest.mark.parametrize("kv_heads,window", [(1, 0), (4, 0), (4, 900)])
def test_tables_of_a_billion_tokens(device, kv_heads, window):
    """A call whose tiles could pass 2^31 by its sizes (128 rows a KV head, 2^30 tokens a table row): the line is counted in units of
    several tiles, whose segments are cut and joined at other places than in a narrow table."""
    g = np.random.default_rng(kv_heads)
    fresh = [60, 64, 0, 4]
    cache, table, lengths, starts = serving(g, [5000, 700, 90, 40], fresh, kv_heads, 16, 64)
    q = g.standard_normal((starts[-1], kv_heads, 64)).astype(np.float32)
    wide = torch.full((4, 1 << 26), -1, dtype=torch.int32, device=device)
    wide[:, :table.shape[1]] = dev(table, device)
    want, far = plain.attend(cache, q, table, lengths.tolist(), starts.tolist(), 0.125, "f32", window=window)
    c, x, n, s = to_device(cache, device), dev(q, device), dev(lengths, device), dev(starts, device)
    for form in (wide, dev(table, device)):
        got = ops.paged_attend(c, x, form, n, s, 0.125, window=window, most=64)
        assert np.all(np.abs(got.double().cpu().numpy() - want) <= far)
