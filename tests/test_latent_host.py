"""The rotation's and the latent cache's entry points without a GPU: what they refuse (nothing is queued), the sizes they ask for, and the
table of angles, which is made on the host."""
import ctypes as C
import math

import pytest
import torch

import latent_plain as plain
from llmp_amd import _lib, ops
from test_paged_host import refused


def cache(**kw):
    base = dict(latent=0x10000, scale=None, rope=0x20000, type=1, pages=8, page=16, width=512, rope_width=64)
    base.update(kw)
    return _lib.LatentCache(**base)


CACHE_REFUSALS = [(dict(latent=None), "null"), (dict(rope=None), "null"), (dict(type=0), "BF16 or F16"), (dict(type=3), "BF16 or F16"), (dict(width=384), "256 or 512"),
                  (dict(rope_width=48), "32 or 64"), (dict(page=8), "pages of"), (dict(page=40), "pages of"), (dict(page=272), "pages of"), (dict(pages=0), "at least one page"),
                  (dict(pages=1 << 27), "2^30"), (dict(latent=0x10008), "16-byte"), (dict(rope=0x20004), "16-byte"), (dict(scale=0x30008), "16-byte")]


# ---------------------------------------------------------------- rotations


def rope(**kw):
    base = dict(x=0x1000, out=0x2000, positions=0x3000, turns=0x4000, tokens=3, x_token_stride=256, x_head_stride=64, out_token_stride=256, out_head_stride=64, type=1, heads=4,
                head_dim=64, first=0, n_dims=64, interleaved=0, inverse=0, magnitude=1.0)
    base.update(kw)
    return _lib.Rope(**base)


@pytest.mark.parametrize("kw,why", [(dict(type=5), "type"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 24), "tokens"), (dict(heads=0), "heads"), (dict(heads=70000), "heads"), (dict(head_dim=0), "channels"),
                                    (dict(n_dims=0), "channels"), (dict(n_dims=63), "channels"), (dict(n_dims=66), "channels"), (dict(first=2), "channels"), (dict(first=-2), "channels"),
                                    (dict(n_dims=1026, head_dim=2048), "channels"), (dict(magnitude=math.nan), "magnitude"), (dict(x=None), "null"), (dict(out=None), "null"),
                                    (dict(positions=None), "null"), (dict(turns=None), "null"), (dict(x=0x1001), "boundaries"), (dict(positions=0x3002), "boundaries"),
                                    (dict(turns=0x4004), "boundaries"), (dict(out=0x1000, out_token_stride=512), "in place"), (dict(out=0x1000, out_head_stride=128), "in place")])
def test_rope_refusals(kw, why):
    refused(_lib.load().llmp_hip_rope(C.byref(rope(**kw)), None), why)


def test_rope_of_nothing():
    lib = _lib.load()
    assert lib.llmp_hip_rope(C.byref(rope(tokens=0, x=None)), None) == 0
    refused(lib.llmp_hip_rope(None, None), "null")


@pytest.mark.parametrize("n_dims,base,options", [(64, 10000.0, {}), (2, 500000.0, {}), (128, 1e6, dict(freq_scale=1 / 40, ext_factor=1.0, corr_dims=(10.0, 23.0))),
                                                 (32, 10000.0, dict(freq_factors=[1.0 + i / 3 for i in range(16)])), (1024, 10000.0, dict(freq_scale=-0.5)), (64, 1e-3, {})])
def test_rope_table(n_dims, base, options):
    """Fractions of a turn to 2^-50 (frequencies to 64-bit floats' 2^-52 of at most 2^10 here, and what comes off whole turns)."""
    got = ops.rope_table(n_dims, base, device="cpu", **options)["turns"]
    want = plain.frequencies(n_dims, base, **options) / (2.0 * math.pi)
    for a, b in zip(got.tolist(), want.tolist()):
        off = ((a % 2 ** 64) / 2 ** 64 - b) % 1.0
        assert min(off, 1.0 - off) <= 2.0 ** -48 * max(abs(b), 1.0)


@pytest.mark.parametrize("args,why", [((0, 1e4, 1.0, 0.0, 0.0, 0.0), "channels"), ((7, 1e4, 1.0, 0.0, 0.0, 0.0), "channels"), ((1026, 1e4, 1.0, 0.0, 0.0, 0.0), "channels"),
                                      ((8, 0.0, 1.0, 0.0, 0.0, 0.0), "positive base"), ((8, -2.0, 1.0, 0.0, 0.0, 0.0), "positive base"), ((8, math.inf, 1.0, 0.0, 0.0, 0.0), "positive base"),
                                      ((8, 1e4, math.nan, 0.0, 0.0, 0.0), "finite"), ((8, 1e4, 1e12, 0.0, 0.0, 0.0), "frequency")])
def test_rope_table_refusals(args, why):
    lib = _lib.load()
    out = (C.c_uint64 * 512)()
    refused(lib.llmp_hip_rope_table(*args, None, out), why)
    refused(lib.llmp_hip_rope_table(8, 1e4, 1.0, 0.0, 0.0, 0.0, None, None), "null")
    for bad in (0.0, math.nan, math.inf):
        refused(lib.llmp_hip_rope_table(8, 1e4, 1.0, 0.0, 0.0, 0.0, (C.c_float * 4)(1.0, bad, 1.0, 1.0), out), "factor 1")


# ---------------------------------------------------------------- the cache


def store(c=None, **kw):
    base = dict(cache=c or cache(), latent=0x1000, rope=0x2000, slots=0x3000, positions=0x4000, turns=0x5000, weight=0x6000, latent_stride=576, rope_stride=576, type=1, tokens=3,
                interleaved=0, eps=1e-6, magnitude=1.0)
    base.update(kw)
    return _lib.LatentStore(**base)


def test_store_and_read_refusals():
    lib = _lib.load()
    read = lambda c=None, slots=0x1000, count=3, kind=1, a=0x2000, b=0x3000: lib.llmp_hip_latent_read(C.byref(c or cache()), slots, count, kind, a, b, None)  # noqa: E731
    for kw, why in CACHE_REFUSALS:
        refused(lib.llmp_hip_latent_store(C.byref(store(cache(**kw))), None), why)
        refused(read(cache(**kw)), why)
    for kw, why in [(dict(latent=None), "null"), (dict(rope=None), "null"), (dict(slots=None), "null"), (dict(type=4), "type"), (dict(tokens=-1), "tokens"), (dict(tokens=(1 << 25) + 1), "tokens"), (dict(latent=0x1008), "16-byte"),
                    (dict(latent_stride=578), "16-byte"), (dict(latent_stride=-576), "16-byte"), (dict(rope=0x2001), "boundaries"), (dict(rope_stride=-64), "boundaries"),
                    (dict(slots=0x3002), "boundaries"), (dict(turns=0x5004), "boundaries"), (dict(positions=0x4001), "boundaries"), (dict(positions=None), "needs positions"),
                    (dict(weight=0x6008), "weight"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps")]:
        refused(lib.llmp_hip_latent_store(C.byref(store(**kw)), None), why)
    assert lib.llmp_hip_latent_store(C.byref(store(tokens=0, latent=None)), None) == 0
    refused(lib.llmp_hip_latent_store(None, None), "null")
    assert read(count=0, slots=None) == 0
    for kw, why in [(dict(slots=None), "slots"), (dict(slots=0x1002), "slots"), (dict(count=-1), "rows"), (dict(count=(1 << 25) + 1), "rows"), (dict(kind=7), "type"), (dict(a=None), "null"),
                    (dict(a=0x2008), "16-byte"), (dict(b=0x3004), "16-byte")]:
        refused(read(**kw), why)
    refused(lib.llmp_hip_latent_read(None, 0x1000, 1, 1, 0x2000, 0x3000, None), "null")


# ---------------------------------------------------------------- the heads' products


def project(**kw):
    base = dict(x=0x1000, w=0x2000, y=0x3000, x_token_stride=512, x_head_stride=128, w_head_stride=128 * 512, w_row_stride=128, y_token_stride=2048, y_head_stride=512, type=1, tokens=3, heads=4,
                k=128, n=512)
    base.update(kw)
    return _lib.LatentProject(**base)


@pytest.mark.parametrize("kw,why", [(dict(type=0), "type"), (dict(k=0), "matrices"), (dict(k=48), "matrices"), (dict(n=16), "matrices"), (dict(n=1 << 17), "matrices"), (dict(heads=0), "heads"),
                                    (dict(heads=70000), "heads"), (dict(tokens=-1), "tokens"), (dict(x=None), "null x"), (dict(w=None), "null w"), (dict(y=None), "null y"), (dict(x=0x1008), "16-byte"),
                                    (dict(w_row_stride=130), "16-byte"), (dict(w_head_stride=-128), "16-byte"), (dict(y_head_stride=516), "16-byte"), (dict(tokens=1 << 24), "tokens")])
def test_project_refusals(kw, why):
    refused(_lib.load().llmp_hip_latent_project(C.byref(project(**kw)), None), why)


def test_project_of_nothing():
    lib = _lib.load()
    assert lib.llmp_hip_latent_project(C.byref(project(tokens=0, x=None)), None) == 0
    refused(lib.llmp_hip_latent_project(None, None), "null")


# ---------------------------------------------------------------- the attentions


def attend(c=None, **kw):
    base = dict(cache=c or cache(), q_latent=0x1000, q_rope=0x2000, out=0x3000, lengths=0x4000, starts=0x5000, table=0x6000, before=None, q_latent_token_stride=2048, q_latent_head_stride=512,
                q_rope_token_stride=768, q_rope_head_stride=192, out_token_stride=2048, out_head_stride=512, table_stride=4, heads=4, requests=2, tokens=3, most_tokens=2, table_width=4, scale=0.1)
    base.update(kw)
    return _lib.LatentAttend(**base)


ATTEND_REFUSALS = [(dict(q_latent=None), "null q_latent"), (dict(q_rope=None), "null q_rope"), (dict(out=None), "null out"), (dict(lengths=None), "null"), (dict(starts=None), "null"),
                   (dict(table=None), "null"), (dict(table=0x6002), "4-byte"), (dict(before=0x7001), "4-byte"), (dict(out=0x3008), "16-byte"), (dict(q_latent_token_stride=2052), "16-byte"),
                   (dict(q_rope_head_stride=-192), "16-byte"), (dict(requests=0), "requests"), (dict(requests=(1 << 24) + 1), "requests"), (dict(tokens=0), "token"), (dict(most_tokens=0), "token"),
                   (dict(heads=0), "heads"), (dict(heads=65536), "heads"), (dict(heads=65535, tokens=1 << 15), "heads"), (dict(table_width=0), "page"), (dict(table_stride=3), "table row"),
                   (dict(table_width=1 << 27, table_stride=1 << 27), "2^30"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale")]


def test_attend_refusals():
    lib = _lib.load()
    for op, why in [(attend(**kw), why) for kw, why in ATTEND_REFUSALS] + [(attend(cache(**kw)), why) for kw, why in CACHE_REFUSALS]:
        assert lib.llmp_hip_latent_attend_scratch(C.byref(op), 256) == 0
        refused(lib.llmp_hip_latent_attend(C.byref(op), 0x100000, 1 << 40, 256, None), why)
    refused(lib.llmp_hip_latent_attend(None, 0x100000, 1 << 40, 256, None), "null")
    for cus in (0, -1, 5000):
        refused(lib.llmp_hip_latent_attend(C.byref(attend()), 0x100000, 1 << 40, cus, None), "compute units")


@pytest.mark.parametrize("kw,rows", [(dict(heads=16, most_tokens=1), 16), (dict(heads=17, most_tokens=1), 128), (dict(heads=4, most_tokens=4, tokens=3), 16), (dict(heads=4, most_tokens=5, tokens=9), 128), (dict(heads=129, most_tokens=1), 128)])
def test_attend_scratch(kw, rows):
    """Two parts a workgroup: whose they are, and a row's maximum, sum and values in F32."""
    lib = _lib.load()
    for width in (256, 512):
        op = attend(cache(width=width), **kw)
        needs = lib.llmp_hip_latent_attend_scratch(C.byref(op), 256)
        groups = 512 if width == 256 and op.most_tokens * op.heads > 128 else 256
        assert needs == 2 * groups * (16 + rows * (8 + 4 * width))
        for scratch, size in ((None, needs), (0x100000, needs - 1), (0x100008, needs)):
            refused(lib.llmp_hip_latent_attend(C.byref(op), scratch, size, 256, None), "scratch")


def prompt(**kw):
    base = dict(q=0x1000, k=0x2000, k_rope=0x3000, v=0x4000, out=0x5000, starts=0x6000, key_starts=None, q_token_stride=768, q_head_stride=192, k_token_stride=1024, k_head_stride=256,
                k_rope_token_stride=576, v_token_stride=1024, v_head_stride=256, out_token_stride=512, out_head_stride=128, type=1, heads=4, requests=2, tokens=3, keys=3, most_tokens=2, nope=128,
                rope_width=64, value=128, scale=0.1)
    base.update(kw)
    return _lib.LatentPrompt(**base)


PROMPT_REFUSALS = [(dict(type=0), "type"), (dict(nope=96, value=96), "heads of"), (dict(nope=128, value=96), "heads of"), (dict(nope=32, value=64), "heads of"), (dict(rope_width=16), "rotated keys"), (dict(heads=0), "heads"),
                   (dict(heads=65536), "heads"), (dict(requests=0), "requests"), (dict(tokens=0), "tokens"), (dict(keys=-1), "keys"), (dict(keys=(1 << 30) + 1), "keys"), (dict(most_tokens=0), "tokens"),
                   (dict(q=None), "null q"), (dict(k=None), "null k"), (dict(v=None), "null v"), (dict(k_rope=None), "null k_rope"), (dict(out=None), "null out"), (dict(starts=None), "I32"),
                   (dict(key_starts=0x7002), "4-byte"), (dict(q=0x1008), "16-byte"), (dict(k_token_stride=1026), "16-byte"), (dict(v_head_stride=-256), "16-byte"), (dict(scale=math.inf), "scale"),
                   (dict(k_token_stride=1 << 24), "2^24"), (dict(v_token_stride=1 << 24), "2^24"), (dict(k_rope_token_stride=1 << 24), "2^24"),
                   (dict(requests=1 << 24, heads=65535, tokens=1 << 20, most_tokens=1 << 20), "too many")]


def test_prompt_refusals():
    lib = _lib.load()
    for kw, why in PROMPT_REFUSALS:
        op = prompt(**kw)
        assert lib.llmp_hip_latent_prompt_scratch(C.byref(op), 256) == 0
        refused(lib.llmp_hip_latent_prompt(C.byref(op), 0x100000, 1 << 40, 256, None), why)
    refused(lib.llmp_hip_latent_prompt(None, 0x100000, 1 << 40, 256, None), "null")
    refused(lib.llmp_hip_latent_prompt(C.byref(prompt()), 0x100000, 1 << 40, 0, None), "compute units")


def test_prompt_scratch():
    """Parts where pairs are cut, 16 bytes where they are taken whole: many rows, or few keys."""
    lib = _lib.load()
    parts = 2 * 512 * (16 + 128 * (8 + 4 * 128))
    for kw, needs in [(dict(), 16), (dict(tokens=8192, keys=8192, most_tokens=8192, heads=64, requests=1), 16), (dict(tokens=1, keys=100000, most_tokens=1, requests=1, key_starts=0x7000), parts),
                      (dict(tokens=300, keys=9000, most_tokens=100, requests=3, key_starts=0x7000), parts),
                      # 1000 prompts of a hundred tokens: whole with a bound on one's, cut where nothing is known of it (25 million blocks else).
                      (dict(tokens=100000, keys=100000, most_tokens=128, heads=32, requests=1000), 16), (dict(tokens=100000, keys=100000, most_tokens=100000, heads=32, requests=1000), parts)]:
        op = prompt(**kw)
        assert lib.llmp_hip_latent_prompt_scratch(C.byref(op), 256) == needs, kw
        for scratch, size in ((None, needs), (0x100000, needs - 1), (0x100008, needs)):
            refused(lib.llmp_hip_latent_prompt(C.byref(op), scratch, size, 256, None), "scratch")


def test_tensors_elsewhere_are_refused():
    """Operands of host memory, or of a device that is not the current one, never reach a launch."""
    x = torch.zeros(2, 2, 64)
    with pytest.raises((AssertionError, RuntimeError)):
        ops.rope(x, torch.zeros(2, dtype=torch.int32), {"turns": torch.zeros(32, dtype=torch.int64), "magnitude": 1.0})
    with pytest.raises((AssertionError, RuntimeError)):
        ops.latent_project(x.bfloat16(), torch.zeros(2, 64, 64, dtype=torch.bfloat16))
