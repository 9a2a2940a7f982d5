"""The attentions over latent vectors where a workgroup has much to do: many requests, many tiles, few workgroups."""
import math

import pytest
import torch

from llmp_amd import ops
from test_gpu_latent import TYPES, check_attend, check_prompt, latent_case, normal

pytestmark = pytest.mark.gpu


def ints(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def test_prompt_of_more_pairs_than_a_launch_has_blocks(device):
    """131072 requests of one token and 128 heads: a row sees its own key alone, and its result is that key's value as it is."""
    requests, heads = 131072, 128
    q, k, v = (torch.randn(requests, heads, d, dtype=torch.bfloat16, device=device) for d in (96, 64, 64))
    k_rope = torch.randn(requests, 32, dtype=torch.bfloat16, device=device)
    got = ops.latent_prompt(q, k, k_rope, v, torch.arange(requests + 1, dtype=torch.int32, device=device), 0.1, most=1)
    assert torch.equal(got, v)


@pytest.mark.parametrize("stride", [1 << 24, (1 << 31) + 8])
def test_prompt_over_one_key_of_any_stride(device, stride):
    """One key as a view of a far larger array's first row, attended by one request's only token: the result is the value."""
    far = torch.randn(3, 64 + 32 + 64, dtype=torch.bfloat16, device=device)
    one = lambda first, last, heads: far[:1, first:last].as_strided((1, heads, last - first), (stride, 0, 1)) if heads else far[:1, first:last].as_strided((1, last - first), (stride, 1))  # noqa: E731
    got = ops.latent_prompt(torch.randn(1, 3, 96, dtype=torch.bfloat16, device=device), one(0, 64, 3), one(64, 96, 0), one(96, 160, 3), ints([0, 1], device), 0.1)
    assert torch.equal(got, far[:1, 96:160].expand(1, 3, 64).reshape(1, 3, 64))


# ---------------------------------------------------------------- many tiles a workgroup: rings go round, page numbers are looked up again, sums are rescaled


def tell_tiles(cache, table, lengths, page, q_latent):
    """Half of the width from its middle on names a token's group of 16 (the queries are zero there): a group that is left out, taken twice or in another's place is
    all of some result, whatever the others are."""
    width = q_latent.shape[2]
    first, groups = width // 2, width // 2
    q_latent[..., first:] = 0.0
    latent = cache["latent"]
    for r, n in enumerate(lengths):
        for p in range(0, n, 16):
            at, count = (int(table[r, p // page]), slice(p % page, p % page + min(16, n - p))), p // 16 % groups
            latent[at][..., first:] = 0
            latent[at][..., first + count] = 0x38 if "scale" in cache else 1.0


def rising(cache, table, lengths, page, q_rope, by):
    """Logits that rise by `by` along every request, so that the running maximum is left behind again and again."""
    q_rope[..., 0] = 16.0
    for r, n in enumerate(lengths):
        for p in range(0, n, page):
            at = int(table[r, p // page])
            count = min(page, n - p)
            cache["rope"][at, :count, 0] = (torch.arange(p, p + count) * (by / max(n, 1) / 16.0)).to(q_rope.dtype)


FORMS = [  # lengths, new tokens, page, heads, most: up to 16 rows a request, 128 rows a workgroup, 32 rows a wave (at width 256)
    ([1, 31, 1025, 2100, 4500], [1, 1, 1, 1, 1], 16, 16, 1), ([4500, 33, 1500], [3, 1, 2], 64, 5, 3), ([31, 4500, 1025], [1, 1, 1], 32, 128, 1), ([1100, 2100], [7, 3], 16, 40, 7),
    ([64, 3001], [1, 2], 128, 130, 2)]


@pytest.mark.parametrize("cus,rise", [(1, 0.0), (1, 100.0), (2, 0.0), (3, 40.0)])
@pytest.mark.parametrize("lengths,new,page,heads,most", FORMS)
@pytest.mark.parametrize("width,rope,dtype,bits", [(512, 64, "bf16", 16), (512, 64, "f16", 8), (256, 32, "f16", 16), (256, 64, "bf16", 8)])
def test_attend_on_few_compute_units(device, monkeypatch, cus, rise, lengths, new, page, heads, most, width, rope, dtype, bits):
    monkeypatch.setattr(ops, "_compute_units", lambda: cus)
    g = torch.Generator().manual_seed(sum(lengths) + heads + width + bits + cus)
    cache, table, starts, q_latent, q_rope = latent_case(g, lengths, new, page, heads, width, rope, dtype, bits)
    scale = (0.2 if bits == 8 else 1.0) / math.sqrt(width + rope)
    tell_tiles(cache, table, lengths, page, q_latent)
    rising(cache, table, lengths, page, q_rope, rise / scale)
    # Pages that are missing, in the first tiles and far behind them.
    for r, n in enumerate(lengths):
        if n > 1024:
            table[r, 2] = -1
            table[r, 1024 // page + 1] = cache["rope"].shape[0] + r
            if page == 16:
                table[r, 90:95] = -1
    check_attend(device, cache, table, lengths, starts, q_latent, q_rope, scale, most=most)


@pytest.mark.parametrize("heads,new,width,bits", [(16, 1, 512, 16), (24, 1, 512, 16), (16, 1, 256, 8), (20, 7, 256, 16)])
def test_attend_over_long_requests(device, heads, new, width, bits):
    """A line of several times what every compute unit takes at least."""
    g = torch.Generator().manual_seed(heads + bits)
    lengths = [30000, 1, 60000, 70, 45000]
    cache, table, starts, q_latent, q_rope = latent_case(g, lengths, [new, 1, 1, 1, 1], 64, heads, width, 64, "bf16", bits)
    scale = (0.2 if bits == 8 else 1.0) / math.sqrt(width + 64)
    tell_tiles(cache, table, lengths, 64, q_latent)
    rising(cache, table, lengths, 64, q_rope, 30.0 / scale)
    check_attend(device, cache, table, lengths, starts, q_latent, q_rope, scale, most=new)


@pytest.mark.parametrize("cus,rise", [(1, 0.0), (4, 100.0), (256, 30.0)])
@pytest.mark.parametrize("new,keys,heads", [([3], [6000], 1), ([140, 1, 30], [1500, 3000, 900], 2)])
@pytest.mark.parametrize("nope,rope,value,dtype", [(128, 64, 128, "bf16"), (64, 32, 64, "f16")])
def test_prompt_on_few_compute_units(device, monkeypatch, cus, rise, new, keys, heads, nope, rope, value, dtype):
    monkeypatch.setattr(ops, "_compute_units", lambda: cus)
    g = torch.Generator().manual_seed(sum(keys) + nope + cus)
    add = lambda v: [sum(v[:i]) for i in range(len(v) + 1)]  # noqa: E731
    starts, key_starts = add(new), add(keys)
    dtype = TYPES[dtype]
    q, k, v = normal(g, starts[-1] + 2, heads, nope + rope, dtype=dtype), normal(g, key_starts[-1], heads, nope, dtype=dtype), normal(g, key_starts[-1], heads, value, dtype=dtype)
    k_rope = normal(g, key_starts[-1], rope, dtype=dtype)
    v[:] = 0.0  # (a group of 16 keys has a dimension: one that is left out or taken twice is all of some result)
    for r in range(len(keys)):
        for j in range(keys[r]):
            v[key_starts[r] + j, :, j // 16 % value] = 1.0
    scale = 1.0 / math.sqrt(nope + rope)
    q[..., nope] = 16.0
    for r, n in enumerate(keys):
        k_rope[key_starts[r]:key_starts[r + 1], 0] = (torch.arange(n) * (rise / scale / n / 16.0)).to(dtype)
    check_prompt(device, q, k, k_rope, v, starts, key_starts, scale, max(new))
