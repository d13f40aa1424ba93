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


def test_outputs_whose_rows_meet(cuda):
    """Rows of an output that share memory are refused; streams and tokens in either order, or between one another, are not."""
    q, kv = torch.randn(3, 2, 64, device=cuda), torch.randn(3, 9, 64, device=cuda)
    weight, slots = torch.ones(64, device=cuda), torch.full((3, 2), -1, dtype=torch.int32, device=cuda)
    pages = ops.PagedKV(torch.randn(1, 3, 16, 64, device=cuda), torch.randn(1, 3, 16, 64, device=cuda),
                        torch.tensor([[0, 0, 1], [3, 1, 2], [5, 2, 0]], dtype=torch.int32, device=cuda), 2)
    for call in (lambda **kw: ops.cross_attn(q, kv, kv, num_heads=1, **kw), lambda **kw: ops.chunk_attn(q, pages, 0, num_heads=1, left=8, **kw),
                 lambda **kw: ops.qk_norm_append(q, kv[:, :2], kv[:, 2:4], pages, 0, slots, num_heads=1, q_weight=weight, **kw)):
        want = call()
        for strides in ((64, 64, 1), (64, 128, 1), (72, 64, 1)):
            with pytest.raises(ValueError, match="rows overlap"):
                call(out=torch.zeros(2000, device=cuda).as_strided((3, 2, 64), strides))
        for strides in ((128, 64, 1), (64, 192, 1), (128, 192, 1), (200, 80, 1)):
            out = torch.zeros(2000, device=cuda).as_strided((3, 2, 64), strides)
            assert call(out=out) is out and torch.equal(out, want)
