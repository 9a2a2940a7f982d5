"""Loads to LDS written as instructions set m0 and say so: the compiler otherwise may keep a value of its own there across them. Needs no GPU and no compiler."""
import glob
import os
import re

SOURCES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llmp_amd", "csrc")


def test_what_sets_m0_says_so():
    """(mxfp8.hip's kernels place every register by hand and are looked at as a whole: tests/test_gemm_named_registers.py.)"""
    found = 0
    for path in sorted(glob.glob(os.path.join(SOURCES, "*.h")) + glob.glob(os.path.join(SOURCES, "*.hip"))):
        if os.path.basename(path) == "mxfp8.hip":
            continue
        with open(path) as f:
            for written in re.findall(r"asm volatile\([^;]*;", f.read()):
                if re.search(r"\bm0, ", written.split('"')[1]):
                    found += 1
                    assert '"m0"' in written.rsplit(":", 1)[1], f"{os.path.basename(path)}: {written}"
    assert found >= 6
