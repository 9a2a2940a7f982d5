"""llmp_hip_paged_attend's weights where one key takes nearly all of a row and its V row is zero, as a first token's often is: what is left of
the output is the other tokens', whose weights the F16 products have to keep."""
import numpy as np
import pytest

import paged_plain as plain
from llmp_amd import ops
from test_gpu_paged import TYPES, dev, rounded, serving, to_device, widened

pytestmark = pytest.mark.gpu


def attend(cache, q, table, length, dtype, scale):
    """(values, how far a kernel's may be from them) of one request's tokens, the last of `length`, in 64 bits. The distance has the
    operator's stated roundings only, each weight's over the V value that it multiplies: the logits' (half a unit of the row's digits
    times sum |k|, 2^-21 of the largest logit for the products and the maximum's subtraction), 2^-20 for exp and the sums; 2^-11 of a
    weight (F32 2^-22) or FLOOR of the row's largest; the result's own type."""
    kv_heads, page, d = cache["k"].shape[1:]
    heads, fresh = q.shape[1], len(q)
    group = heads // kv_heads
    at = table[0, :plain.ceil(length, page)]
    k, v = plain.values(cache, at)
    k, v = (np.swapaxes(x, 0, 1).reshape(kv_heads, -1, d)[:, :length] for x in (k, v))
    vs = np.repeat(cache["v_scale"][at].astype(np.float64), page, axis=0)[:length]
    digit, weight = (8355584.0, 2.0 ** -22) if dtype == "f32" else (32639.0, 2.0 ** -11)
    last = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    out, far = np.zeros(q.shape), np.zeros(q.shape)
    for t in range(fresh):
        end = length - fresh + t + 1
        for h in range(heads):
            x, kk, vv, ss = q[t, h].astype(np.float64), k[h // group, :end], v[h // group, :end], vs[:end, h // group]
            s = kk @ x * scale
            e = scale * np.abs(x).max() / digit / 2 * np.abs(kk).sum(1).max() + 2.0 ** -21 * np.abs(s).max() + 2.0 ** -20
            w = np.exp(s - s.max())
            total, largest = w.sum(), (w * ss).max()
            out[t, h] = w @ vv / total
            codes = np.abs(vv) / ss[:, None]
            far[t, h] = ((2 * e + weight) * (w @ np.abs(vv)) + FLOOR[dtype] * largest * codes.sum(0)) / total + last * np.abs(out[t, h])
            if dtype == "f16":
                far[t, h] += 2.0 ** -25
    return out, far


FLOOR = {"f32": 2.0 ** -46, "bf16": 2.0 ** -35, "f16": 2.0 ** -35}


def dominated(g, length, fresh, kv_heads, page, d, nats, alike):
    """A request whose first key is `nats` above the others for a query of ones in dimension 0, its V row zero, the other V rows positive
    (what is lost of many weights adds up). `alike`: the other keys are one, so their weights and what they lose are."""
    cache, table, lengths, starts = serving(g, [length], [fresh], kv_heads, page, d)
    cache["k"][:] = 0 if alike else g.integers(-4, 5, cache["k"].shape)
    cache["k"][..., 0] = 0
    cache["k_scale"][:] = 0.25
    cache["v"][:] = g.integers(20, 128, cache["v"].shape)
    cache["v_scale"][:] = 0.01
    first = table[0, 0]
    cache["k"][first, :, 0, :] = 0
    cache["k"][first, :, 0, 0] = 4 * nats
    cache["v"][first, :, :, 0] = 0
    return cache, table, lengths, starts


def check(device, dtype, length, fresh, kv_heads, page, d, nats, alike):
    g = np.random.default_rng(length + fresh + nats)
    cache, table, lengths, starts = dominated(g, length, fresh, kv_heads, page, d, nats, alike)
    q = np.zeros((fresh, 2 * kv_heads, d)) if alike else g.standard_normal((fresh, 2 * kv_heads, d)) * 0.1
    q[..., 0] = 1.0
    qt, q = rounded(q, dtype)
    want, far = attend(cache, q, table, length, dtype, 1.0)
    assert (far <= 0.03 * want).all()  # (an output of zeros, or of tenths lost, is far outside)
    c, qt, n, s = to_device(cache, device), qt.to(device), dev(lengths, device), dev(starts, device)
    assert qt.dtype is TYPES[dtype]
    for form in (table, widened(table, cache, fresh, fresh, 2 * kv_heads)):
        got = ops.paged_attend(c, qt, dev(form, device), n, s, 1.0).double().cpu().numpy()
        wrong = ~(np.abs(got - want) <= far)
        assert not wrong.any(), f"{form.shape[1]} pages a row: {int(wrong.sum())} of {wrong.size} too far off, up to {np.max(np.abs(got - want) / far)} of the distance"


SHAPES = [(4000, 1, 2, 64, 128), (3001, 40, 1, 16, 64), (2500, 70, 1, 32, 256), (7000, 5, 1, 128, 128)]


@pytest.mark.parametrize("alike", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("length,fresh,kv_heads,page,d", SHAPES)
def test_a_dominating_token_leaves_the_others_their_weights(device, dtype, length, fresh, kv_heads, page, d, alike):
    for nats in (12, 18):
        check(device, dtype, length, fresh, kv_heads, page, d, nats, alike)


@pytest.mark.parametrize("alike", [True, False])
@pytest.mark.parametrize("length,fresh,kv_heads,page,d", SHAPES)
def test_f32_keeps_what_an_f16_leaves_of_a_weight(device, length, fresh, kv_heads, page, d, alike):
    for nats in (12, 16, 20):
        check(device, "f32", length, fresh, kv_heads, page, d, nats, alike)
