"""The build's check of the waits over latent rows (llmp_amd/csrc/check_counted_waits.py) sees a tile of which a path asks for a part only, and a wait for part of one.
(tests/test_counted_waits.py runs the check over the sources themselves.)"""
import importlib.util
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def module():
    spec = importlib.util.spec_from_file_location("check_counted_waits", os.path.join(ROOT, "llmp_amd", "csrc", "check_counted_waits.py"))
    loaded = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(loaded)
    return loaded


LOAD, WAIT = "\t;;#ASMSTART\n\tglobal_load_lds_dwordx4 v1, s[0:1]\n\t;;#ASMEND", "\t;;#ASMSTART\n\ts_waitcnt vmcnt(%d)\n\t;;#ASMEND"


def body(before, loop, waits=(6, 3)):
    """`before` loads, then a loop of `loop` loads on one path and none on the other, with waits of both numbers."""
    return "\n".join([LOAD] * before + [".LBB0_1:", "\ts_cbranch_scc0 .LBB0_2", WAIT % waits[0], "\ts_branch .LBB0_3", ".LBB0_2:", WAIT % waits[1], ".LBB0_3:", "\ts_barrier",
                                        "\ts_cbranch_vccz .LBB0_4"] + [LOAD] * loop + [".LBB0_4:", "\tglobal_load_dword v2, v3, off", "\ts_cbranch_scc1 .LBB0_1", WAIT % 0, "\ts_endpgm"])


@pytest.mark.parametrize("before,loop,waits,holds", [(9, 3, (6, 3), True), (6, 6, (6, 3), True), (9, 2, (6, 3), False), (8, 3, (6, 3), False), (9, 3, (5, 3), False), (9, 4, (6, 3), False)])
def test_a_tile_of_too_few_or_too_many_loads_is_found(module, before, loop, waits, holds):
    if holds:
        assert module.check_tiles("kernel", body(before, loop, waits)) == 3
    else:
        with pytest.raises(AssertionError, match="part of a tile|whole tiles"):
            module.check_tiles("kernel", body(before, loop, waits))


def test_a_load_of_the_compilers_among_those_counted_is_found(module):
    with pytest.raises(AssertionError, match="compiler's own"):
        module.check_tiles("kernel", body(9, 3).replace(LOAD, "\tglobal_load_lds_dwordx4 v1, s[0:1]"))
    assert module.check_tiles("kernel", body(5, 2, (0, 0))) is None  # nothing is counted where every wait is for all


def test_the_checks_flags_are_the_builds(module):
    with open(os.path.join(ROOT, "llmp_amd", "csrc", "Makefile")) as f:
        made = {m.group(1): m.group(2).split() for m in re.finditer(r"^build/(\S+)\.o: FLAGS \+= (.*)$", f.read(), re.M)}
    assert made == module.FLAGS
