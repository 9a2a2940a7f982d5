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


def test_strides_of_one_key_are_not_looked_at():
    """A single key's rows lie wherever they lie: what its token stride says is not used (a view of one row out of a larger array has any)."""
    lib = _lib.load()
    for stride in (1 << 24, 1 << 40, -8, 3):
        far = dict(k_token_stride=stride, v_token_stride=stride, k_rope_token_stride=stride)
        assert lib.llmp_hip_latent_prompt_scratch(C.byref(prompt(tokens=1, keys=1, requests=1, most_tokens=1, **far)), 256) > 0
        assert lib.llmp_hip_latent_prompt_scratch(C.byref(prompt(tokens=1, keys=0, requests=1, most_tokens=1, **far)), 256) > 0
        assert lib.llmp_hip_latent_prompt_scratch(C.byref(prompt(tokens=1, keys=2, requests=1, most_tokens=1, key_starts=0x7000, **far)), 256) == 0
