"""What the paged cache's entry points refuse, and the scratch they ask for, beyond tests/test_paged_host.py."""
import ctypes as C

from llmp_amd import _lib
from test_paged_host import attend, refused, select


def test_before_lies_at_a_4_byte_boundary():
    lib = _lib.load()
    refused(lib.llmp_hip_paged_attend(C.byref(attend(before=0x7002)), 0x100000, 1 << 40, 256, None), "4-byte")
    refused(lib.llmp_hip_paged_select(C.byref(select(before=0x7002)), 0x100000, 1 << 40, None), "4-byte")
    assert lib.llmp_hip_paged_attend_scratch(C.byref(attend(before=0x7000)), 256) == lib.llmp_hip_paged_attend_scratch(C.byref(attend()), 256) > 0
    assert lib.llmp_hip_paged_select_scratch(C.byref(select(before=0x7000))) == lib.llmp_hip_paged_select_scratch(C.byref(select())) > 0
