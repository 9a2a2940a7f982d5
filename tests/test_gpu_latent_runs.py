"""The attentions over latent vectors where a workgroup has much to do: many requests, many tiles, few workgroups."""
import torch

import pytest

from llmp_amd import ops

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
