"""Batch tables on the GPU: page steps against the host pool and a plain model, K/V
append through a slot map bit for bit, adapter plans against a stable sort.  All
values are whole numbers or copies: every comparison is exact."""

import numpy as np
import pytest
import torch

from parakeet_amd import _lib, ops
from parakeet_amd.pool import DevicePagePool, PagePool
from tests._tables_model import RaggedPool, plan_model

pytestmark = pytest.mark.gpu


def _up(a, cuda, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).to(cuda)


def _same_pool(pool, model):
    assert pool.free_list().tolist() == list(model.free)
    A, ring = pool.state.appended.cpu().numpy(), pool.state.ring.cpu().numpy()
    assert A.tolist() == model.A
    np.testing.assert_array_equal(ring, np.stack([model.ring(s) for s in range(len(model.A))]))


@pytest.mark.parametrize("left,chunk,P,slots,extra", [(70, 2, 16, 9, 0), (70, 14, 16, 7, 5), (5, 1, 4, 5, 1), (9, 3, 2, 7, 0), (0, 2, 4, 3, 2), (40, 5, 64, 4, 0)])
def test_steps_match_the_host_pool(cuda, left, chunk, P, slots, extra):
    rng = np.random.default_rng(left * 7 + chunk + P)
    M = (left + chunk + P - 2) // P + 1
    order = rng.permutation(slots * M + extra)
    host = PagePool(slots, P, left, chunk, num_pages=len(order), page_order=order)
    dev = DevicePagePool(slots, P, left, chunk, cuda, num_pages=len(order), page_order=order)
    assert dev.max_pages == host.max_pages
    for step in range(120):
        if rng.random() < 0.15:
            gone = rng.permutation(slots)[: rng.integers(1, slots + 1)]
            for s in gone:
                host.reset_slot(int(s))
            dev.reset_slots(gone)
        batch = rng.permutation(slots)[: rng.integers(0, slots + 1)].astype(np.int32)
        rows, place = dev.advance(batch)
        want = host.advance(batch)
        np.testing.assert_array_equal(rows.cpu().numpy(), want)
        pos = want[:, :1] + np.arange(chunk)
        np.testing.assert_array_equal(place.cpu().numpy(), np.take_along_axis(want[:, 1:], pos // P % M, 1) * P + pos % P)
    assert dev.free_list().tolist() == host.free_list().tolist() and dev.free_pages() == host.free_pages()
    for s in range(slots):
        a, ring = host.slot_info(s)
        b, got = dev.slot_info(s)
        assert a == b and ring.tolist() == got.tolist()
    host.reset_all()
    dev.reset_all()
    assert dev.free_list().tolist() == host.free_list().tolist()


@pytest.mark.parametrize("n,slots,left,chunk,P", [(1, 1, 70, 2, 16), (63, 70, 20, 7, 8), (64, 64, 70, 14, 16), (257, 300, 70, 2, 16), (1025, 1100, 16, 5, 4),
                                                  (2049, 2500, 70, 2, 8), (5000, 5000, 300, 14, 16)])
def test_ragged_steps_match_the_model(cuda, n, slots, left, chunk, P):
    rng = np.random.default_rng(n)
    dev = DevicePagePool(slots, P, left, chunk, cuda)
    order = rng.permutation(dev.num_pages)
    dev = DevicePagePool(slots, P, left, chunk, cuda, page_order=order)
    model = RaggedPool(slots, P, left, chunk, order)
    for step in range(30 if n < 2000 else 12):
        batch = rng.permutation(slots)[:n].astype(np.int32)
        lengths = rng.integers(0, chunk + 1, n)
        if step % 3 == 1:  # what a caller may leave in: too long, negative, absent, named twice
            lengths[rng.integers(0, n)] = chunk + 5
            lengths[rng.integers(0, n)] = -3
            batch[rng.integers(0, n)] = slots
            batch[rng.integers(0, n)] = -1
            batch[rng.integers(0, n)] = batch[rng.integers(0, n)]
        rows, place = dev.advance(_up(batch, cuda), _up(lengths, cuda))
        want_rows, want_place = model.advance(batch.tolist(), lengths.tolist())
        np.testing.assert_array_equal(rows.cpu().numpy(), want_rows)
        np.testing.assert_array_equal(place.cpu().numpy(), want_place)
        if step % 4 == 3:
            gone = rng.integers(-1, slots + 1, 1 + n // 10)
            dev.reset_slots(_up(gone, cuda))
            model.reset(gone.tolist())
    _same_pool(dev, model)


def test_the_most_slots(cuda):
    """Every slot of the largest pool in one step, twice, against array arithmetic."""
    S, P, left, chunk = _lib.PAGE_STEP_MAX_SLOTS, 16, 14, 9
    dev = DevicePagePool(S, P, left, chunk, cuda)
    rng = np.random.default_rng(2)
    A, taken = np.zeros(S, dtype=np.int64), 0
    first = None
    for step in range(2):
        slots, lengths = rng.permutation(S), rng.integers(0, chunk + 1, S)
        rows, place = (t.cpu().numpy() for t in dev.advance(_up(slots, cuda), _up(lengths, cuda)))
        a = A[slots]
        np.testing.assert_array_equal(rows[:, 0], a)
        # no window has moved past a page yet: pages come in order of the streams
        need = (a + lengths + P - 1) // P - (a + P - 1) // P
        at = taken + np.cumsum(need) - need
        if step == 0:
            np.testing.assert_array_equal(rows[:, 1], np.where(need > 0, at, -1))
            first = np.full(S, -1)
            first[slots] = rows[:, 1]
        else:
            old = np.where(first[slots] >= 0, first[slots], np.where(need > 0, at, -1))
            np.testing.assert_array_equal(rows[:, 1], old)
            np.testing.assert_array_equal(rows[:, 2], np.where(a + lengths > P, at + need - 1, -1))
        t = np.arange(chunk)[None, :]
        pos = a[:, None] + t
        want = np.take_along_axis(rows[:, 1:], pos // P % dev.max_pages, 1) * P + pos % P
        np.testing.assert_array_equal(place, np.where(t < lengths[:, None], want, -1))
        taken += int(need.sum())
        A[slots] = a + lengths
    assert dev.free_pages() == dev.num_pages - taken
    assert dev.state.head.tolist() == [taken % dev.num_pages, dev.num_pages - taken]


def test_every_slot_the_same(cuda):
    dev = DevicePagePool(3, 16, 70, 2, cuda)
    rows, place = dev.advance(_up(np.full(3000, 1), cuda))
    assert rows[0, :2].tolist() == [0, 0] and place[0].tolist() == [0, 1]
    assert (rows[1:, 0] == 0).all() and (rows[1:, 1:] == -1).all() and (place[1:] == -1).all()
    assert dev.slot_info(1)[0] == 2 and dev.free_pages() == dev.num_pages - 1


@pytest.mark.parametrize("n", [5, 17, 63, 64, 66, 1001, 3500, 4100])
def test_every_slot_named_twice(cuda, n):
    """n streams, the second half naming the slots of the first in another order: the
    second half is absent, wherever in the batch its first mention is."""
    slots, left, chunk, P = n, 20, 7, 8
    dev = DevicePagePool(slots, P, left, chunk, cuda)
    model = RaggedPool(slots, P, left, chunk, np.arange(dev.num_pages))
    rng = np.random.default_rng(n)
    for _ in range(5):
        once = rng.permutation(slots)[: (n + 1) // 2]
        batch = np.concatenate([once, rng.permutation(once)])[:n].astype(np.int32)
        lengths = rng.integers(0, chunk + 1, n)
        rows, place = dev.advance(_up(batch, cuda), _up(lengths, cuda))
        want_rows, want_place = model.advance(batch.tolist(), lengths.tolist())
        np.testing.assert_array_equal(rows.cpu().numpy(), want_rows)
        np.testing.assert_array_equal(place.cpu().numpy(), want_place)
    _same_pool(dev, model)


def test_positions_past_2_30(cuda):
    dev = DevicePagePool(2, 16, 70, 2, cuda)
    dev.state.appended.fill_(2**31 - 20)
    k = (2**31 - 20 - 72) // 16
    dev.state.ring.copy_(torch.tensor([[(k + (r - k) % 6) % 6 + 6 * s for r in range(6)] for s in range(2)], dtype=torch.int32))
    before = dev.state.ring.clone()
    rows, place = dev.advance([1, 0], _up([1, 2], cuda))
    assert rows[:, 0].tolist() == [2**31 - 20] * 2
    r = (2**31 - 20) // 16 % 6  # frames 12 and 13 of a page that is held
    assert place.tolist() == [[int(before[1, r]) * 16 + 12, -1], [int(before[0, r]) * 16 + 12, int(before[0, r]) * 16 + 13]]
    assert dev.state.appended.tolist() == [2**31 - 18, 2**31 - 19]


def test_step_in_a_graph_and_on_another_stream(cuda):
    dev, host = DevicePagePool(20, 16, 70, 14, cuda), PagePool(20, 16, 70, 14)
    slots = _up(np.arange(20), cuda)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        rows, place = dev.advance(slots)
    torch.cuda.current_stream(cuda).wait_stream(side)
    np.testing.assert_array_equal(rows.cpu().numpy(), host.advance(np.arange(20)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows, place = dev.advance(slots)
    for step in range(12):
        batch = np.random.default_rng(step).permutation(20).astype(np.int32)
        slots.copy_(torch.from_numpy(batch))
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(rows.cpu().numpy(), host.advance(batch))
        if step % 5 == 0:
            dev.reset_slot(3)
            host.reset_slot(3)
    assert dev.free_list().tolist() == host.free_list().tolist()


# ---------------------------------------------------------------------------


def _fill(shape, dtype, cuda, seed):
    return torch.randn(shape, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,P", [(512, 16), (640, 8), (72, 32), (8, 1), (1024, 64)])
def test_append_by_slot_map(cuda, dtype, D, P):
    rng = np.random.default_rng(D + P)
    Ly, N, B, T = 3, 11, 5, 7
    k_pool, v_pool = _fill((Ly, N, P, D), dtype, cuda, 1), _fill((Ly, N, P, D), dtype, cuda, 2)
    qkv = _fill((B, T, 3 * D), dtype, cuda, 3)
    places = rng.permutation(N * P)[: min(B * T, N * P)]
    m = np.full(B * T, -1)
    m[rng.permutation(B * T)[: len(places)]] = places
    m[rng.integers(0, B * T, 4)] = [-1, N * P, 2**31 - 1, -(2**31)]  # padding, and places that no page holds
    m = m.reshape(B, T)
    want = []
    for pool, part in ((k_pool, 1), (v_pool, 2)):
        w = ops.page_blocks(pool).clone()
        for b in range(B):
            for t in range(T):
                if 0 <= m[b, t] < N * P:
                    w[1, m[b, t] // P, :, m[b, t] % P] = qkv[b, t, part * D : (part + 1) * D].view(w.shape[2], w.shape[4])
        want.append(w)
    pages = ops.PagedKV(k_pool, v_pool, torch.zeros(B, 2, dtype=torch.int32, device=cuda), 1)
    wide = torch.full((B, T + 3), 0, dtype=torch.int32, device=cuda)  # the map as a view of wider rows
    wide[:, :T] = _up(m, cuda)
    copies = [p.clone() for p in (k_pool, v_pool)]
    ops.kv_append_slots(pages, 1, qkv[..., D : 2 * D], qkv[..., 2 * D :], wide[:, :T])
    assert torch.equal(ops.page_blocks(k_pool), want[0]) and torch.equal(ops.page_blocks(v_pool), want[1])
    # packed rows, the ones behind the last stream left out
    k_pool.copy_(copies[0])
    v_pool.copy_(copies[1])
    flat = m.reshape(-1)
    keep = np.flatnonzero((flat >= 0) & (flat < N * P))
    rows = qkv.reshape(-1, 3 * D)[_up(keep, cuda, np.int64)]
    rows = torch.cat([rows, torch.full((3, 3 * D), float("nan"), dtype=dtype, device=cuda)])
    packed = _up(np.concatenate([flat[keep], [-1] * 3]), cuda)
    ops.kv_append_slots(pages, 1, rows[:, D : 2 * D], rows[:, 2 * D :], packed)
    assert torch.equal(ops.page_blocks(k_pool), want[0]) and torch.equal(ops.page_blocks(v_pool), want[1])
    ops.kv_append_slots(pages, 1, rows[:0, :D], rows[:0, :D], packed[:0])  # nothing to write
    assert torch.equal(ops.page_blocks(k_pool), want[0])


def test_append_checks_devices_and_layers(cuda):
    pool = torch.zeros(1, 2, 16, 64, dtype=torch.float16, device=cuda)
    pages = ops.PagedKV(pool, pool.clone(), torch.zeros(1, 3, dtype=torch.int32, device=cuda), 2)
    kv, m = torch.zeros(4, 64, dtype=torch.float16, device=cuda), torch.zeros(4, dtype=torch.int32, device=cuda)
    with pytest.raises(RuntimeError, match="layer 1"):
        ops.kv_append_slots(pages, 1, kv, kv, m)
    with pytest.raises(ValueError, match="devices"):
        ops.kv_append_slots(pages, 0, kv, kv, m.cpu())
    with pytest.raises(RuntimeError, match="aligned"):
        odd = torch.zeros(4 * 64 + 4, dtype=torch.float16, device=cuda)[4:].view(4, 64)
        ops.kv_append_slots(pages, 0, odd, kv, m)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_ragged_streams_end_in_the_windows(cuda, dtype):
    """page_step -> kv_append_slots -> kv_gather: each stream's window is its own frames,
    however its chunks were cut."""
    rng = np.random.default_rng(5)
    left, chunk, P, D, S = 21, 6, 4, 64, 9
    pool = DevicePagePool(S, P, left, chunk, cuda, page_order=rng.permutation(S * 8))
    assert pool.num_pages == S * pool.max_pages
    nan = lambda: torch.full((1, pool.num_pages, P, D), float("nan"), dtype=dtype, device=cuda)  # noqa: E731
    k_pool, v_pool = nan(), nan()
    said = [np.zeros((0, 2 * D), np.float32) for _ in range(S)]
    for step in range(25):
        slots = rng.permutation(S)[: rng.integers(1, S + 1)]
        lengths = rng.integers(0, chunk + 1, len(slots))
        kv = rng.standard_normal((len(slots), chunk, 2 * D)).astype(np.float16).astype(np.float32)
        rows, place = pool.advance(_up(slots, cuda), _up(lengths, cuda))
        t = torch.from_numpy(kv).to(cuda).to(dtype)
        pages = ops.PagedKV(k_pool, v_pool, rows, pool.max_pages)
        if step % 2:
            ops.kv_append_slots(pages, 0, t[..., :D], t[..., D:], place)
        else:
            keep = place.reshape(-1) >= 0
            ops.kv_append_slots(pages, 0, t[..., :D].reshape(-1, D)[keep], t[..., D:].reshape(-1, D)[keep], place.reshape(-1)[keep])
        for i, s in enumerate(slots):
            said[s] = np.concatenate([said[s], kv[i, : lengths[i]]])
        # the window that the step's attention reads: the frames before the step
        k, v = ops.kv_gather(pages, 0, len(slots), left, 0)
        for i, s in enumerate(slots):
            was = said[s][: len(said[s]) - lengths[i]][-left:]
            want = np.concatenate([np.zeros((left - len(was), 2 * D), np.float32), was])
            np.testing.assert_array_equal(torch.cat([k[i], v[i]], -1).float().cpu().numpy(), want)


# ---------------------------------------------------------------------------


@pytest.mark.parametrize("B,T,G", [(1, 1, 1), (7, 3, 5), (64, 2, 64), (65, 14, 3), (1000, 2, 512), (1023, 1, 200), (3001, 7, 31), (4096, 14, 1), (20000, 1, 512)])
@pytest.mark.parametrize("how", ["even", "skewed", "none", "one"])
def test_plan(cuda, B, T, G, how):
    rng = np.random.default_rng(B + G)
    ids = {
        "even": rng.integers(-2, G + 2, B),
        "skewed": np.minimum(rng.geometric(0.3, B) - 2, G + 1),
        "none": np.where(rng.random(B) < 0.5, -1, G),
        "one": np.full(B, G - 1),
    }[how]
    if how == "none":
        ids[0] = -(2**31)
    p = ops.adapter_plan(_up(ids, cuda), T, num_adapters=G)
    order, sorted_ids, tiles = plan_model(ids.astype(np.int64), T, G)
    np.testing.assert_array_equal(p.order.cpu().numpy(), order)
    np.testing.assert_array_equal(p.ids.cpu().numpy(), sorted_ids)
    np.testing.assert_array_equal(p.tiles.cpu().numpy(), tiles)


def test_plan_of_no_streams(cuda):
    p = ops.adapter_plan(torch.zeros(0, dtype=torch.int32, device=cuda), 2, num_adapters=4)
    assert p.order.shape == (0,) and p.ids.shape == (0,) and p.tiles.shape == (0, 4)
    with pytest.raises(RuntimeError, match="up to 512"):
        ops.adapter_plan(torch.zeros(1, dtype=torch.int32, device=cuda), 2, num_adapters=513)
