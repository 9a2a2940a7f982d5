"""Attention over latent vectors where values are infinite or no numbers: what a row sees of them is in its result as the definition has it, the sum of weight * value,
whatever its place in a tile and whatever else the tile holds."""
import math

import pytest
import torch

from llmp_amd import ops
from test_gpu_latent import TYPES, normal

pytestmark = pytest.mark.gpu


def ints(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def bits(t):
    return t.contiguous().view(torch.int16)


# ---------------------------------------------------------------- the expanded form

# (key, dimension, value): sums of one sign stay infinite, of both, or of a NaN, become none. The first tile of a request is one that not all rows see.
BAD = [(0, 3, math.inf), (9, 3, math.inf), (1, 8, -math.inf), (20, 11, math.inf), (33, 11, -math.inf), (40, 17, math.nan), (70, 20, -math.inf), (135, 25, math.inf), (290, 30, math.inf),
       (291, 33, -math.inf), (298, 33, math.inf), (299, 38, math.nan)]


@pytest.mark.parametrize("new,heads", [(300, 2), (40, 3), (1, 5), (200, 128)])
@pytest.mark.parametrize("dtype,nope,rope,value,more", [("bf16", 128, 64, 128, 0), ("f16", 64, 32, 64, 0), ("f16", 128, 32, 64, 2500), ("bf16", 64, 64, 128, 2500)])
def test_prompt_values_that_rows_see(device, dtype, nope, rope, value, more, new, heads):
    """Weights here are within 2^14 of each other, so that none becomes zero: a dimension's sum is what its values' signs say, the other dimensions have the bits that they have
    without. (With `more` keys in front the keys are cut into runs.)"""
    g = torch.Generator().manual_seed(new + heads + nope)
    keys = 300 + more
    q, k = normal(g, new, heads, nope + rope, dtype=TYPES[dtype]), normal(g, keys, heads, nope, dtype=TYPES[dtype])
    v, k_rope = normal(g, keys, heads, value, dtype=TYPES[dtype]), normal(g, keys, rope, dtype=TYPES[dtype])

    def run():
        return ops.latent_prompt(q.to(device), k.to(device), k_rope.to(device), v.to(device), ints([0, new], device), 0.05, key_starts=ints([0, keys], device), most=new).cpu()

    clean = run()
    want = torch.zeros(new, value)
    sees = torch.arange(keys - new, keys)
    for key, dim, bad in BAD:
        v[more + key, :, dim] = bad
        want[:, dim] += torch.where(sees >= more + key, torch.tensor(bad), torch.tensor(0.0))
    got = run()
    odd = ~torch.isfinite(want)
    assert odd.any()
    for h in range(heads):
        assert torch.equal(bits(got[:, h])[~odd], bits(clean[:, h])[~odd]), h
        assert torch.equal(got[:, h].float().nan_to_num(nan=7.0)[odd], want.nan_to_num(nan=7.0)[odd]), h


@pytest.mark.parametrize("more", [0, 2500])
def test_prompt_infinities_of_no_weight(device, more):
    """A logit of minus infinity: the weight is zero, so that a value changes nothing where it is finite, and is no number where it is infinite."""
    g = torch.Generator().manual_seed(5)
    new, heads, keys = 130, 2, 130 + more
    q, k = normal(g, new, heads, 192, dtype=torch.bfloat16), normal(g, keys, heads, 128, dtype=torch.bfloat16)
    v, k_rope = normal(g, keys, heads, 128, dtype=torch.bfloat16), normal(g, keys, 64, dtype=torch.bfloat16)
    q[..., 1] = -q[..., 1].abs() - 0.5
    bad = [more + 2, more + 50, more + 100, more + 129]
    k[bad, :, 1] = math.inf

    def run():
        return ops.latent_prompt(q.to(device), k.to(device), k_rope.to(device), v.to(device), ints([0, new], device), 0.05, key_starts=ints([0, keys], device), most=new).cpu()

    clean = run()
    assert torch.isfinite(clean.float()).all()
    for i, key in enumerate(bad):
        v[key, :, 10 * i] = math.inf
    got = run()
    odd = torch.zeros(new, 128, dtype=torch.bool)
    for i, key in enumerate(bad):
        odd[key - more:, 10 * i] = True
    for h in range(heads):
        assert torch.isnan(got[:, h].float()[odd]).all() and torch.equal(bits(got[:, h])[~odd], bits(clean[:, h])[~odd])
