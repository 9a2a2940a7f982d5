"""The paged cache's entry points without a GPU: what they refuse (nothing is queued), and the sizes they ask for."""
import ctypes as C

import pytest

from llmp_amd import _lib


def cache(**kw):
    base = dict(k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000, low=0x50000, high=0x60000, pages=8, kv_heads=2, page=16, head_dim=64)
    base.update(kw)
    return _lib.PagedCache(**base)


CACHE_REFUSALS = [(dict(k=None), "null"), (dict(v_scale=None), "null"), (dict(low=None), "low and high"), (dict(head_dim=96), "head sizes"),
                  (dict(page=8), "pages of"), (dict(page=40), "pages of"), (dict(page=272), "pages of"), (dict(pages=0), "at least one page"),
                  (dict(kv_heads=0), "KV heads"), (dict(kv_heads=70000), "KV heads"), (dict(v=0x20008), "16-byte")]


def refused(code, why):
    assert code == 1 and why in _lib.load().llmp_hip_last_error().decode(), _lib.load().llmp_hip_last_error()


def plan(**kw):
    base = dict(before=0x1000, after=0x2000, table=0x3000, ring=0x4000, counters_in=0x5000, counters=0x5000, starts=0x6000, lengths=0x7000,
                slots=0x8000, positions=0x9000, owners=0xA000, work=0xB000, scratch=0xC000, table_stride=4, requests=3, table_width=4, ring_size=8,
                page=16, tokens=5, work_items=5)
    base.update(kw)
    return _lib.PagedPlan(**base)


@pytest.mark.parametrize("kw,why", [(dict(requests=0), "requests"), (dict(ring_size=0), "ring"), (dict(table_width=0), "table"), (dict(tokens=-1), "tokens"),
                                    (dict(page=0), "pages"), (dict(before=None), "null"), (dict(slots=None), "null"), (dict(work=None), "null"),
                                    (dict(scratch=None), "null"), (dict(table_stride=3), "table row"), (dict(work=0xB004), "at 16"),
                                    (dict(lengths=0x7002), "4-byte"), (dict(work_items=4), "work items")])
def test_plan_refusals(kw, why):
    refused(_lib.load().llmp_hip_paged_plan(C.byref(plan(**kw)), None), why)


def test_work_items_cover_every_split_of_the_tokens():
    """All ways of giving a few tokens to a few requests, at every place in a page: never more touched pages than said."""
    lib = _lib.load()
    for page in (1, 2, 3, 4):
        for tokens in range(0, 9):
            most = 0
            for first in range(tokens + 1):
                for a in range(page):
                    for b in range(page):
                        touched = sum((o + n - 1) // page + 1 for o, n in ((a, first), (b, tokens - first)) if n)
                        most = max(most, touched)
            assert most <= lib.llmp_hip_paged_work_items(2, tokens, page) <= tokens
    assert lib.llmp_hip_paged_plan_scratch(0) == 0 and lib.llmp_hip_paged_plan_scratch(7) >= 3 * 8 * 4


def store(c=None, **kw):
    base = dict(cache=c or cache(), k=0x1000, v=0x2000, work=0x3000, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64, type=0,
                tokens=3, work_items=2)
    base.update(kw)
    return _lib.PagedStore(**base)


def test_store_and_read_refusals():
    lib = _lib.load()
    for kw, why in CACHE_REFUSALS:
        refused(lib.llmp_hip_paged_store(C.byref(store(cache(**kw))), None), why)
        refused(lib.llmp_hip_paged_read(C.byref(cache(**kw)), 0x1000, 1, 2, 0, 0x2000, 0x3000, None), why)
    for kw, why in [(dict(type=3), "type"), (dict(k=None), "null k"), (dict(v=0x2004), "16-byte"), (dict(k_token_stride=130), "16-byte"), (dict(work=None), "work items"),
                    (dict(work=0x3008), "work items"), (dict(tokens=-1), "tokens"), (dict(type=1, v_head_stride=68), "16-byte")]:
        refused(lib.llmp_hip_paged_store(C.byref(store(**kw)), None), why)
    assert lib.llmp_hip_paged_store(C.byref(store(tokens=0, k=None)), None) == 0  # nothing to do: nothing queued
    refused(lib.llmp_hip_paged_store(None, None), "null")
    refused(lib.llmp_hip_paged_read(C.byref(cache()), None, 1, 2, 0, 0x2000, 0x3000, None), "page numbers")
    refused(lib.llmp_hip_paged_read(C.byref(cache()), 0x1000, 1, 2, 5, 0x2000, 0x3000, None), "type")
    refused(lib.llmp_hip_paged_read(C.byref(cache()), 0x1000, 1, 2, 0, 0x2008, 0x3000, None), "16-byte")
    refused(lib.llmp_hip_paged_read(C.byref(cache()), 0x1000, -1, 2, 0, 0x2000, 0x3000, None), "pages every")


def attend(c=None, **kw):
    base = dict(cache=c or cache(), q=0x1000, out=0x2000, lengths=0x3000, starts=0x4000, table=0x5000, lists=None, sinks=None, q_token_stride=256, q_head_stride=64,
                out_token_stride=256, out_head_stride=64, table_stride=4, type=0, heads=4, requests=2, tokens=3, most_tokens=2, table_width=4,
                list_pages=0, window=0, scale=0.125, softcap=0.0)
    base.update(kw)
    return _lib.PagedAttend(**base)


@pytest.mark.parametrize("kw,why", [(dict(heads=5), "query heads"), (dict(q=None), "null q"), (dict(out=0x2004), "16-byte"), (dict(type=7), "type"),
                                    (dict(requests=0), "requests"), (dict(tokens=0), "token"), (dict(most_tokens=0), "token"), (dict(table_width=0), "page"),
                                    (dict(table_stride=3), "table row"), (dict(lengths=None), "null"), (dict(table=0x5002), "4-byte"),
                                    (dict(lists=0x6000, list_pages=0), "lists"), (dict(table_width=1 << 27, table_stride=1 << 27), "2^30"), (dict(window=-1), "window"),
                                    (dict(scale=float("inf")), "scale"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"),
                                    (dict(q_token_stride=-64), "16-byte")])
def test_attend_refusals(kw, why):
    lib = _lib.load()
    op = attend(**kw)
    assert lib.llmp_hip_paged_attend_scratch(C.byref(op), 256) == 0
    refused(lib.llmp_hip_paged_attend(C.byref(op), 0x100000, 1 << 40, 256, None), why)


def test_attend_cache_and_scratch():
    lib = _lib.load()
    for kw, why in CACHE_REFUSALS:
        refused(lib.llmp_hip_paged_attend(C.byref(attend(cache(**kw))), 0x100000, 1 << 40, 256, None), why)
    assert lib.llmp_hip_paged_attend_scratch(C.byref(attend(cache(low=None, high=None))), 256) > 0
    needs = lib.llmp_hip_paged_attend_scratch(C.byref(attend()), 256)
    for scratch, size in ((None, needs), (0x100000, needs - 1), (0x100008, needs)):
        refused(lib.llmp_hip_paged_attend(C.byref(attend()), scratch, size, 256, None), "scratch")


def select(c=None, **kw):
    base = dict(cache=c or cache(), q=0x1000, lengths=0x3000, starts=0x4000, table=0x5000, lists=0x6000, q_token_stride=256, q_head_stride=64, table_stride=4, type=1,
                heads=4, requests=2, tokens=3, most_tokens=2, table_width=4, keep=3, first=1, recent=1)
    base.update(kw)
    return _lib.PagedSelect(**base)


@pytest.mark.parametrize("kw,why", [(dict(c=cache(low=None, high=None)), "needed here"), (dict(heads=3), "query heads"), (dict(keep=0), "pages"), (dict(keep=5000), "pages"),
                                    (dict(first=2, recent=2), "pages"), (dict(first=-1), "pages"), (dict(lists=None), "null"), (dict(type=9), "type"),
                                    (dict(tokens=0), "token"), (dict(table_stride=1), "table row"), (dict(table_width=1 << 27, table_stride=1 << 27), "2^30")])
def test_select_refusals(kw, why):
    lib = _lib.load()
    op = select(**kw)
    assert lib.llmp_hip_paged_select_scratch(C.byref(op)) == 0
    refused(lib.llmp_hip_paged_select(C.byref(op), 0x100000, 1 << 40, None), why)
    good = select()
    needs = lib.llmp_hip_paged_select_scratch(C.byref(good))
    assert needs == 3 * 2 * 4 * 4
    refused(lib.llmp_hip_paged_select(C.byref(good), 0x100000, needs - 1, None), "scratch")
