"""The attentions over latent vectors at the ends of what they take, without a GPU: calls of more workgroups than a launch has are cut otherwise."""
import ctypes as C

import pytest

from llmp_amd import _lib
from test_latent_host import prompt

PARTS = 2 * 512 * (16 + 128 * (8 + 4 * 128))  # of a call whose pairs are cut, on 256 compute units


@pytest.mark.parametrize("requests,heads,new,needs", [(131072, 128, 1, PARTS), (131072, 127, 1, 16), (1 << 20, 16, 1, PARTS), (1 << 19, 16, 1, 16), (100000, 100, 129, PARTS), (1 << 20, 2000, 1, PARTS),
                                                     ((1 << 24) // 16 - 1, 16, 1, 16), (1 << 24, 1, 1, PARTS), ((1 << 24) - 8, 1, 1, 16)])
def test_prompts_of_more_pairs_than_a_launch_has_blocks(requests, heads, new, needs):
    """A launch has less than 2^32 threads, 256 a pair that is taken whole: 2^24 - 8 of them, by eights, at most."""
    op = prompt(requests=requests, heads=heads, tokens=requests * new, keys=requests * new, most_tokens=new)
    assert _lib.load().llmp_hip_latent_prompt_scratch(C.byref(op), 256) == needs
