"""What a text decoder's calls refuse and what they take, on the GPU."""

import pytest
import torch

from parakeet_amd import ops

pytestmark = pytest.mark.gpu


def test_pages_are_copied_under_autocast(cuda):
    """A copy has no type to change: under autocast it is what it is without."""
    k = torch.randn(2, 4, 16, 64, device=cuda)
    v, want = -k, k.clone()
    moves = ops.PageMoves(torch.tensor([[3, 1]], dtype=torch.int32, device=cuda), torch.ones(1, dtype=torch.int32, device=cuda))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        ops.kv_move_pages(k, v, moves)
    want[:, 1] = want[:, 3]
    assert torch.equal(k, want) and torch.equal(v, -want)


def test_pools_with_gradients(cuda):
    """Pools that need a gradient are refused, but under no_grad, where the same bits come out."""
    g = torch.Generator(device=cuda).manual_seed(0)
    k, v = (torch.randn(1, 4, 16, 64, generator=g, device=cuda) for _ in range(2))
    rows = torch.tensor([[40, 2, 0, 3]], dtype=torch.int32, device=cuda)
    q = torch.randn(1, 3, 64, generator=g, device=cuda)
    call = lambda k, v: ops.chunk_attn(q, ops.PagedKV(k, v, rows, 3), 0, num_heads=1, left=20)  # noqa: E731
    want, leaf = call(k, v), v.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        call(k, leaf)
    with torch.no_grad():
        assert torch.equal(call(k, leaf), want)
