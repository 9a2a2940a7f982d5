"""Workspaces that a caller gives (`scratch`): memory that a kernel may not write, or not all of, is refused before a launch."""
import gc

import pytest
import torch

from llmp_amd import ops


def calls(device, scratch):
    """Every wrapper that takes a workspace, on small operands."""
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    paged, latent = ops.paged_cache(4, 2, 16, 64, device=device), ops.latent_cache(4, 16, 256, 32, device=device)
    zeros = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device=device)  # noqa: E731
    table, lengths, starts = ints([[0, 1]]), ints([5]), ints([0, 1])
    cells = zeros(256 * 34 * 2, dtype=torch.uint8)
    return [lambda: ops.attn_vec_quant(ops.TYPE_Q8_0, zeros(2, 1, 64, dtype=torch.float32), cells, cells, zeros(1, 256, dtype=torch.float16), 64, 2, 1, 256, 0.1, scratch=scratch),
            lambda: ops.paged_attend(paged, zeros(1, 4, 64), table, lengths, starts, 0.1, scratch=scratch),
            lambda: ops.paged_select(paged, zeros(1, 4, 64), table, lengths, starts, 2, scratch=scratch),
            lambda: ops.latent_attend(latent, zeros(1, 4, 256), zeros(1, 4, 32), table, lengths, starts, 0.1, scratch=scratch),
            lambda: ops.latent_prompt(zeros(1, 4, 96), zeros(1, 4, 64), zeros(1, 32), zeros(1, 4, 64), starts, 0.1, scratch=scratch)]


def test_workspaces_of_host_memory():
    like = torch.zeros(4)
    assert ops._workspace(None, 100, like).nbytes == 100 and ops._workspace(None, 3, like).nbytes == 16
    with pytest.raises(AssertionError, match="workspace"):
        ops._workspace(torch.zeros(1 << 20, dtype=torch.uint8), 100, like)


@pytest.fixture
def nothing_left():
    """Refusals hold the frames they came from, and so the tensors, until they are collected: not in a later test that counts memory."""
    yield
    gc.collect()


@pytest.mark.gpu
def test_workspaces_are_looked_at(device, nothing_left):
    for scratch in (torch.zeros(64 << 20, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8, device=device).expand(64 << 20), torch.zeros(128 << 20, dtype=torch.uint8, device=device)[::2]):
        for call in calls(device, scratch):
            with pytest.raises(AssertionError, match="workspace"):
                call()
    for call, plain in zip(calls(device, torch.zeros(32 << 20, dtype=torch.float32, device=device)), calls(device, None)):
        assert torch.equal(call(), plain())
