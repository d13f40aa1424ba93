"""Page steps whose caller reads the rows alone: no slot map is written, everything else is
as with one; and resets, which read no lengths."""

import ctypes

import numpy as np
import pytest
import torch

from parakeet_amd import _lib, ops
from parakeet_amd.modules.cache import ModelCache
from parakeet_amd.pool import DevicePagePool

pytestmark = pytest.mark.gpu


def _same(a, b):
    for name in ("queue", "head", "appended", "ring"):
        assert torch.equal(getattr(a.state, name), getattr(b.state, name)), name


@pytest.mark.parametrize("n,slots", [(1, 1), (64, 70), (65, 65), (3500, 3600), (3501, 4000)])
def test_rows_without_places(cuda, n, slots):
    rng = np.random.default_rng(n)
    pools = [DevicePagePool(slots, 8, 20, 5, cuda) for _ in range(2)]
    for _ in range(9):
        batch = torch.from_numpy(rng.permutation(slots)[:n].astype(np.int32)).to(cuda)
        lengths = torch.from_numpy(rng.integers(0, 6, n).astype(np.int32)).to(cuda)
        rows, place = pools[0].advance(batch, lengths)
        got, none = pools[1].advance(batch, lengths, places=False)
        assert none is None and place is not None and torch.equal(rows, got)
    _same(*pools)
    given = torch.empty(n, 5, dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="without places"):
        pools[1].advance(batch, lengths, slot_map=given, places=False)
    _same(*pools)


def test_cache_steps_write_no_places(cuda, monkeypatch):
    """The cache's own reader of a step, the attention, takes the rows."""
    maps = []
    real = ops.page_step
    monkeypatch.setattr(ops, "page_step", lambda *a, **kw: maps.append(real(*a, **kw)[1]))
    cache = ModelCache(1, [20, 4], 64, 9, batch_size=3, device=cuda, dtype=torch.float16, device_pages=True)
    kv = torch.zeros(3, 5, 64, dtype=torch.float16, device=cuda)
    cache.update_attn_cache(0, kv, kv)
    assert maps == [None]


def test_reset_reads_no_lengths(cuda):
    """What a caller leaves in the step's other fields changes nothing in a reset."""
    pools = [DevicePagePool(5, 8, 20, 5, cuda) for _ in range(2)]
    batch = torch.tensor([3, 1, 4], dtype=torch.int32, device=cuda)
    for pool in pools:
        for _ in range(4):
            pool.advance(batch)
    gone = torch.tensor([4, 1], dtype=torch.int32, device=cuda)
    pools[0].reset_slots(gone)
    a, dev, _, _ = pools[1].state._args(gone)
    lengths = torch.tensor([5, -7], dtype=torch.int32, device=cuda)
    a.reset, a.lengths, a.rows_stride, a.slot_map_stride = 1, lengths.data_ptr(), -1, -1
    _lib.check(_lib.lib().pk_page_step(ctypes.byref(a), ops._stream(dev)), "pk_page_step")
    _same(*pools)
    assert pools[1].slot_info(4)[0] == 0 and pools[1].slot_info(3)[0] == 20
