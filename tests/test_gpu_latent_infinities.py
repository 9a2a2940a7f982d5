"""Attention over latent vectors where values are infinite or no numbers: what a row sees of them is in its result as the definition has it, the sum of weight * value,
whatever its place in a tile and whatever else the tile holds."""
import math

import pytest
import torch

import latent_plain as plain
from llmp_amd import ops
from test_gpu_latent import TYPES, latent_case, normal

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


# ---------------------------------------------------------------- the absorbed form


@pytest.mark.parametrize("width,dtype", [(512, "bf16"), (256, "f16"), (512, "f16"), (256, "bf16")])
@pytest.mark.parametrize("heads,new,at", [(8, 2, 75), (5, 3, 75), (16, 1, 75), (16, 1, 89), (3, 5, 86), (48, 33, 75), (40, 3, 70), (128, 1, 89), (128, 2, 75), (20, 60, 64), (160, 3, 87)])
def test_infinities_of_no_weight(device, width, dtype, heads, new, at):
    """A token of infinities whose logit is minus infinity for all: no number in those dimensions of the rows that see it, and nothing anywhere else; and so whatever the later
    tokens hold that a row does not see, which are cleaned out of the same tile."""
    g = torch.Generator().manual_seed(width + heads + at)
    cache, table, starts, q_latent, q_rope = latent_case(g, [90], [new], 16, heads, width, 64, dtype, 16)
    q_latent[..., 5], q_latent[..., 131] = -q_latent[..., 5].abs() - 0.5, -q_latent[..., 131].abs() - 0.5
    latent = cache["latent"]

    def run():
        on = {k: v.to(device) for k, v in cache.items()}
        return ops.latent_attend(on, q_latent.to(device), q_rope.to(device), table.to(device), ints([90], device), ints(starts, device), 0.02, most=new).cpu()[:new]

    def where(p):
        return int(table[0, p // 16]), p % 16

    latent[where(at)] = 0.0
    latent[where(at)][5], latent[where(at)][131] = math.inf, math.inf
    first = run()
    sees = (torch.arange(90 - new, 90) >= at)[:, None, None].expand(-1, heads, width)
    odd = sees & torch.isin(torch.arange(width), torch.tensor([5, 131]))[None, None]
    assert torch.equal(torch.isnan(first.float()), odd) and torch.isfinite(first.float()[~odd]).all()
    # The same but for the last token, which the rows of the last new token see alone.
    if at != 89 and new > 1:
        for bad in (math.nan, math.inf):
            latent[where(89)][::3] = bad
            again = run()
            assert torch.equal(bits(again[:-1]), bits(first[:-1]))
    # The other dimensions are as without the token: its weight is zero.
    latent[where(at)] = 0.0
    latent[where(89)][::3] = latent[where(89)].nan_to_num(0.0, 0.0, 0.0)[::3]
    entries = table[0, :6].long()
    c = latent.double()[entries].reshape(-1, width)[:90]
    k = torch.cat([c, cache["rope"].double()[entries].reshape(-1, 64)[:90]], 1)
    q = torch.cat([q_latent[:new], q_rope[:new]], -1).double().reshape(new * heads, -1)
    want, size, logits = plain.attention(q, k, c, 0.02, (90 - new + torch.arange(new)).repeat_interleave(heads), torch.arange(90) != at)
    rows = slice(0, new * heads if at == 89 or new == 1 else (new - 1) * heads)  # (the last token's own values were others)
    got = torch.where(odd, 0.0, first.float()).reshape(new * heads, width)
    want, size = torch.where(odd.reshape(new * heads, width), 0.0, want), torch.where(odd.reshape(new * heads, width), 0.0, size)
    plain.close(got[rows], want[rows], size[rows], logits[rows], TYPES[dtype], width + 64, 90)


@pytest.mark.parametrize("heads,new", [(16, 1), (40, 3)])
def test_rows_of_no_logit_but_minus_infinity(device, heads, new):
    """They are as rows that see nothing: zeros (but where an infinity of the absorbed form's own rows is seen)."""
    g = torch.Generator().manual_seed(heads)
    cache, table, starts, q_latent, q_rope = latent_case(g, [50], [new], 16, heads, 512, 64, "bf16", 16)
    q_rope[..., 3] = -2.0
    for p in range(50):
        cache["rope"][int(table[0, p // 16]), p % 16, 3] = math.inf
    on = {k: v.to(device) for k, v in cache.items()}
    got = ops.latent_attend(on, q_latent.to(device), q_rope.to(device), table.to(device), ints([50], device), ints(starts, device), 0.02, most=new)
    assert (got[:new] == 0).all()
    q, k, v, k_rope = (normal(g, *s, dtype=torch.bfloat16) for s in ((new, 2, 192), (50, 2, 128), (50, 2, 128), (50, 64)))
    q[..., 130], k_rope[:, 2] = -2.0, math.inf
    got = ops.latent_prompt(q.to(device), k.to(device), k_rope.to(device), v.to(device), ints([0, new], device), 0.05, key_starts=ints([0, 50], device), most=new)
    assert (got == 0).all()
