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
