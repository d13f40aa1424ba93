"""What a text decoder's calls refuse, on the CPU: pools that something follows, outputs whose rows meet, scales past
fp32, slots past 32 bits."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from parakeet_amd import _lib, ops
from parakeet_amd.pool import DevicePagePool


class _Marked(torch.Tensor):
    pass


def _pool_calls():
    z = lambda *s: torch.zeros(s)  # noqa: E731
    rows, slots = torch.zeros(2, 7, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    moves = ops.PageMoves(torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    return {
        "qk_norm_append": lambda k, v: ops.qk_norm_append(z(2, 3, 256), z(2, 3, 128), z(2, 3, 128), ops.PagedKV(k, v, rows, 6), 0, slots, num_heads=4),
        "chunk_attn": lambda k, v: ops.chunk_attn(z(2, 3, 256), ops.PagedKV(k, v, rows, 6), 0, num_heads=4, left=9),
        "kv_move_pages": lambda k, v: ops.kv_move_pages(k, v, moves),
    }


@pytest.mark.parametrize("name", ["qk_norm_append", "chunk_attn", "kv_move_pages"])
@pytest.mark.parametrize("which", [0, 1])
def test_pools_that_something_follows(name, which):
    call = _pool_calls()[name]
    pools = [torch.zeros(1, 8, 16, 128) for _ in range(2)]
    other = lambda t: [t if i == which else p for i, p in enumerate(pools)]  # noqa: E731
    leaf = torch.zeros(1, 8, 16, 128, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward pass"):
        call(*other(leaf))
    with torch.no_grad(), pytest.raises(RuntimeError, match="HIP device"):
        call(*other(leaf))
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        call(*other(forward_ad.make_dual(leaf.detach(), torch.ones_like(leaf))))
    with pytest.raises(RuntimeError, match="plain tensors"):
        call(*other(leaf.detach().as_subclass(_Marked)))
    with pytest.raises(RuntimeError, match="HIP device"):
        call(*pools)


# strides of out [3, 2, 64] and whether rows of it meet
@pytest.mark.parametrize("strides,meet", [
    ((128, 64, 1), False), ((64, 192, 1), False), ((64, 64, 1), True), ((64, 128, 1), True), ((128, 128, 1), True), ((192, 64, 1), False),
    ((128, 320, 1), False), ((64, 136, 1), True), ((128, 192, 1), False), ((72, 64, 1), True), ((256, 72, 1), False),
])
def test_outputs_whose_rows_meet(strides, meet):
    cells = torch.zeros(3, 2, 64)
    idx = torch.arange(3)[:, None, None] * strides[0] + torch.arange(2)[None, :, None] * strides[1] + torch.arange(64)
    assert (idx.unique().numel() < cells.numel()) == meet
    out = torch.zeros(2000).as_strided((3, 2, 64), strides)
    call = lambda: ops._head_out("chunk_attn", out, torch.zeros(3, 2, 64), out.device, [])  # noqa: E731
    if meet:
        with pytest.raises(ValueError, match="rows overlap"):
            call()
    else:
        assert call() is out


def test_outputs_of_many_rows():
    """Neither stride is a multiple of the other's rows: still told apart."""
    query = torch.zeros(5, 7, 64)
    for sb in range(64, 1200, 64):
        for st in range(64, 1200, 64):
            out = torch.zeros(20000).as_strided((5, 7, 64), (sb, st, 1))
            at = (torch.arange(5)[:, None] * sb + torch.arange(7) * st).flatten()
            meet = at.unique().numel() < 35
            try:
                ops._head_out("cross_attn", out, query, out.device, [])
                assert not meet, (sb, st)
            except ValueError:
                assert meet, (sb, st)


@pytest.mark.parametrize("name,make", [("pk_chunk_attn", _lib.ChunkAttnArgs), ("pk_cross_attn", _lib.CrossAttnArgs)])
@pytest.mark.parametrize("scale,ok", [(2.0e38, True), (2.4e38, False), (3.4e38, False), (1e-45, True)])
def test_scales_at_the_ends_of_fp32(name, make, scale, ok):
    """Scores are counted in powers of two: the scale times log2 e has to be finite, too. An empty batch asks no more."""
    memory = (ctypes.c_char * 4096)()
    at = ctypes.addressof(memory) + 15 & ~15
    a = make()
    a.device, a.batch, a.chunk, a.num_heads, a.head_dim, a.scale = -1, 0, 1, 1, 64, scale
    if make is _lib.ChunkAttnArgs:
        L = a.pages
        L.k_pool = L.v_pool = L.rows = at
        L.num_layers, L.num_pages, L.page_size, L.d_model, L.rows_stride, L.max_pages = 1, 1, 16, 64, 2, 1
    else:
        a.kv_heads, a.states = 1, 1
    rc = getattr(_lib.lib(), name)(ctypes.byref(a), None)
    assert rc == (_lib.PK_OK if ok else _lib.PK_ERR_INVALID), _lib.last_error()
    assert ok or "scale" in _lib.last_error()


@pytest.mark.parametrize("src,dst", [([0], [2**32 + 1]), ([0], [-(2**32) + 1]), ([2**32], [1])])
def test_slots_past_32_bits(src, dst):
    with pytest.raises(ValueError, match="slots must be"):
        DevicePagePool(4, 16, 70, 2, "cpu").fork(src, dst)
