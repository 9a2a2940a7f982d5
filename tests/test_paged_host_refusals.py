"""What the paged cache's entry points refuse, and the scratch they ask for, beyond tests/test_paged_host.py."""
import ctypes as C

import pytest
import torch

from llmp_amd import _lib, ops
from test_paged_host import attend, cache, plan, refused, select, store


def test_before_lies_at_a_4_byte_boundary():
    lib = _lib.load()
    refused(lib.llmp_hip_paged_attend(C.byref(attend(before=0x7002)), 0x100000, 1 << 40, 256, None), "4-byte")
    refused(lib.llmp_hip_paged_select(C.byref(select(before=0x7002)), 0x100000, 1 << 40, None), "4-byte")
    assert lib.llmp_hip_paged_attend_scratch(C.byref(attend(before=0x7000)), 256) == lib.llmp_hip_paged_attend_scratch(C.byref(attend()), 256) > 0
    assert lib.llmp_hip_paged_select_scratch(C.byref(select(before=0x7000))) == lib.llmp_hip_paged_select_scratch(C.byref(select())) > 0


def test_scratch_of_a_selection_is_its_scores_where_they_go_through_memory():
    lib = _lib.load()
    wide = dict(table_width=4096, table_stride=4096, keep=4096, tokens=2048, most_tokens=2048, requests=8)
    for kw, needs in [(dict(wide), 16),  # every page is chosen: no scores
                      (dict(wide, keep=64, requests=1, table_width=200, table_stride=200), 16),  # one launch, the scores in LDS
                      (dict(wide, keep=64), 2048 * 2 * 4096 * 4),  # a row of keys is more than LDS takes
                      (dict(wide, keep=64, tokens=2, most_tokens=1, requests=2), 2 * 2 * 4096 * 4)]:  # few workgroups: two launches
        op = select(heads=4, **kw)
        assert lib.llmp_hip_paged_select_scratch(C.byref(op)) == needs, kw
        for scratch, size in ((None, needs), (0x100000, needs - 1), (0x100008, needs)):
            refused(lib.llmp_hip_paged_select(C.byref(op), scratch, size, None), "scratch")


def test_plans_of_more_outputs_than_an_int_steps_through():
    lib = _lib.load()
    for kw in (dict(tokens=(1 << 30) + 1, work_items=1 << 30), dict(work_items=(1 << 30) + 1), dict(ring_size=(1 << 31) - 1)):
        refused(lib.llmp_hip_paged_plan(C.byref(plan(**kw)), None), "2^30")


def test_tables_of_more_tokens_and_heads_than_an_int_counts_tiles_of():
    lib = _lib.load()
    wide = dict(table_width=1 << 26, table_stride=1 << 26)
    for kv_heads, good in ((64, True), (65, False), (128, False)):
        op = attend(cache(kv_heads=kv_heads), heads=kv_heads, **wide)
        assert (lib.llmp_hip_paged_attend_scratch(C.byref(op), 256) > 0) == good
    refused(lib.llmp_hip_paged_attend(C.byref(op), 0x100000, 1 << 40, 256, None), "2^36")


def test_strides_of_one_token_or_one_head_are_not_looked_at():
    lib = _lib.load()
    one = dict(tokens=1, most_tokens=1, requests=1)
    assert lib.llmp_hip_paged_attend_scratch(C.byref(attend(q_token_stride=257, out_token_stride=1, **one)), 256) > 0
    assert lib.llmp_hip_paged_select_scratch(C.byref(select(q_token_stride=257, **one))) > 0
    assert lib.llmp_hip_paged_attend_scratch(C.byref(attend(cache(kv_heads=1), heads=1, q_head_stride=1, out_head_stride=-1)), 256) > 0
    refused(lib.llmp_hip_paged_attend(C.byref(attend(q_head_stride=65, **one)), 0x100000, 1 << 40, 256, None), "16-byte")
    refused(lib.llmp_hip_paged_store(C.byref(store(cache(kv_heads=1), tokens=2, k_token_stride=65, k_head_stride=1)), None), "16-byte")


def test_the_wrappers_take_no_host_memory():
    """A tensor in host memory would be an address that no kernel may read: refused before anything is asked of the GPU."""
    host = ops.paged_cache(4, 2, 16, 64, device="cpu")
    ints = [torch.zeros(n, dtype=torch.int32) for n in (2, 2, 8, 3, 3)]
    q, table = torch.zeros(2, 4, 64), torch.zeros((2, 2), dtype=torch.int32)
    work = torch.zeros((2, 4), dtype=torch.int32)
    for call in (lambda: ops.paged_plan(ints[0], ints[1], table, ints[2], ints[3], 16, 2),
                 lambda: ops.paged_store(host, q[:, :2], q[:, :2], work),
                 lambda: ops.paged_read(host, ints[0]),
                 lambda: ops.paged_attend(host, q, table, ints[0], ints[3], 0.125),
                 lambda: ops.paged_select(host, q, table, ints[0], ints[3], 2)):
        with pytest.raises(AssertionError, match="GPU"):
            call()
