"""Forks, compaction and page copies of a device page pool against a plain model, entry for
entry: whole numbers and copies, every comparison exact."""

import numpy as np
import pytest
import torch

from parakeet_amd import _lib, ops
from parakeet_amd.modules import ModelCache
from parakeet_amd.pool import DevicePagePool
from tests._page_moves_model import compact, fork
from tests._tables_model import RaggedPool

pytestmark = pytest.mark.gpu


def _up(a, cuda):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(cuda)


def _same(pool, model):
    assert pool.free_list().tolist() == list(model.free)
    assert pool.state.appended.tolist() == model.A
    np.testing.assert_array_equal(pool.state.ring.cpu().numpy(), np.stack([model.ring(s) for s in range(len(model.A))]))


def _moves(moves):
    n = int(moves.count)
    pairs = moves.pairs.cpu().numpy()
    assert (pairs[n:] == -1).all()
    return [tuple(p) for p in pairs[:n].tolist()]


@pytest.mark.parametrize("slots,left,chunk,P,extra", [(7, 70, 2, 16, 0), (40, 20, 7, 8, 13), (300, 70, 14, 16, 0), (9, 700, 5, 4, 3), (1, 5, 1, 4, 0),
                                                      (600, 300, 14, 16, 5), (700, 3, 2, 1, 50)])
def test_forks_and_compaction_match_the_model(cuda, slots, left, chunk, P, extra):
    """Steps, forks with bad and repeated slots, resets and compactions in turn: small pools in one launch, large ones in several."""
    rng = np.random.default_rng(slots + left)
    pages = slots * ((left + chunk + P - 2) // P + 1) + extra
    order = rng.permutation(pages)
    dev = DevicePagePool(slots, P, left, chunk, cuda, num_pages=pages, page_order=order)
    model = RaggedPool(slots, P, left, chunk, order)
    for turn in range(24):
        for _ in range(int(rng.integers(1, 12))):
            batch = rng.permutation(slots)[: rng.integers(1, slots + 1)].astype(np.int32)
            lengths = rng.integers(0, chunk + 1, len(batch))
            rows, place = dev.advance(_up(batch, cuda), _up(lengths, cuda))
            want = model.advance(batch.tolist(), lengths.tolist())
        np.testing.assert_array_equal(rows.cpu().numpy(), want[0])
        np.testing.assert_array_equal(place.cpu().numpy(), want[1])
        n = int(rng.integers(0, slots + 1))
        src, dst = rng.integers(0, slots, n), rng.integers(0, slots, n)
        if turn % 3 == 0:  # as a caller does: distinct, apart
            both = rng.permutation(slots)
            n = int(rng.integers(0, slots // 2 + 1))
            src, dst = rng.choice(both[n:], n), both[:n]
        elif turn % 3 == 1 and n:
            src[rng.integers(0, n)], dst[rng.integers(0, n)] = slots, -1
        assert _moves(ops.page_fork(dev.state, _up(src, cuda), _up(dst, cuda))) == fork(model, src.tolist(), dst.tolist())
        _same(dev, model)
        if turn % 4 == 1:
            gone = rng.integers(0, slots, 1 + slots // 3)
            dev.reset_slots(_up(gone, cuda))
            model.reset(gone.tolist())
        if turn % 2:
            assert _moves(dev.compact()) == compact(model, pages)
            _same(dev, model)


def test_a_full_pool_forks(cuda):
    """Every page held: the pages that the destinations give back are the ones that are taken."""
    dev, model = DevicePagePool(4, 4, 6, 2, cuda), RaggedPool(4, 4, 6, 2, range(12))
    assert dev.num_pages == 12
    for _ in range(5):
        dev.advance([0, 1, 2, 3])
        model.advance([0, 1, 2, 3], [2] * 4)
    assert dev.free_pages() == len(model.free)
    assert _moves(dev.fork([0, 0], [3, 1])) == fork(model, [0, 0], [3, 1])
    _same(dev, model)
    assert _moves(dev.compact()) == compact(model, 12)
    _same(dev, model)


def test_the_most_slots(cuda):
    """The largest pool: half of the slots forked into the other half, compacted after every third is freed."""
    S, P, left, chunk = _lib.PAGE_STEP_MAX_SLOTS, 16, 14, 9
    dev, model = DevicePagePool(S, P, left, chunk, cuda), RaggedPool(S, P, left, chunk, range(S * 3))
    rng = np.random.default_rng(3)
    both = rng.permutation(S)
    lengths = rng.integers(0, chunk + 1, S)
    dev.advance(_up(both, cuda), _up(lengths, cuda))
    model.advance(both.tolist(), lengths.tolist())
    src, dst = both[: S // 2], both[S // 2 :]
    assert _moves(ops.page_fork(dev.state, _up(src, cuda), _up(dst, cuda))) == fork(model, src.tolist(), dst.tolist())
    gone = np.arange(0, S, 3)
    dev.reset_slots(_up(gone, cuda))
    model.reset(gone.tolist())
    assert _moves(dev.compact()) == compact(model, S * 3)
    _same(dev, model)


def test_every_destination_twice(cuda):
    S = 3000
    dev, model = DevicePagePool(2 * S, 4, 6, 2, cuda), RaggedPool(2 * S, 4, 6, 2, range(2 * S * 3))
    assert dev.max_pages == 3
    dev.advance(_up(np.arange(2 * S), cuda))
    model.advance(list(range(2 * S)), [2] * (2 * S))
    rng = np.random.default_rng(5)
    src = rng.integers(0, S, 2 * S)
    dst = np.concatenate([S + rng.permutation(S), S + rng.permutation(S)])
    assert _moves(ops.page_fork(dev.state, _up(src, cuda), _up(dst, cuda))) == fork(model, src.tolist(), dst.tolist())
    _same(dev, model)


def test_nothing_to_move(cuda):
    dev = DevicePagePool(5, 16, 70, 2, cuda)
    assert _moves(dev.compact()) == [] and dev.free_list().tolist() == list(range(dev.num_pages))
    assert _moves(dev.fork([], [])) == []
    dev.advance([2])
    assert _moves(dev.fork([0], [3])) == []  # a stream without frames
    assert _moves(dev.fork([0], [2])) == [] and dev.slot_info(2)[0] == 0 and dev.free_pages() == dev.num_pages
    k = torch.randn(2, dev.num_pages, 16, 32, device=cuda)
    v, kept = k.clone(), k.clone()
    ops.kv_move_pages(k, v, dev.compact())
    ops.kv_move_pages(k, v, dev.fork([], []))
    assert torch.equal(k, kept) and torch.equal(v, kept)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Ly,N,P,D", [(1, 9, 16, 512), (3, 50, 8, 72), (24, 20, 16, 1024), (2, 6, 1, 8), (2, 30, 64, 1000)])
def test_copies(cuda, dtype, Ly, N, P, D):
    """Pages of all layers copied as the moves say, nothing else; pairs out of range and behind the count left out."""
    g = torch.Generator().manual_seed(N)
    k, v = (torch.randn(Ly, N, P, D, generator=g).to(dtype) for _ in range(2))
    perm = torch.randperm(N, generator=g)
    n = N // 2
    pairs = torch.stack([perm[:n], perm[N - n :]], 1)
    pairs = torch.cat([pairs, torch.tensor([[N, 0], [0, -1], [-1, 1]]), torch.tensor([[1, 2]])]).int()
    dk, dv = k.to(cuda), v.to(cuda)
    ops.kv_move_pages(dk, dv, ops.PageMoves(pairs.to(cuda), torch.tensor([n + 3], dtype=torch.int32, device=cuda)))
    for x in (k, v):
        x[:, pairs[:n, 1].long()] = x[:, pairs[:n, 0].long()]
    assert torch.equal(dk.cpu(), k) and torch.equal(dv.cpu(), v)
    ops.kv_move_pages(dk, dv, ops.PageMoves(pairs.to(cuda), torch.tensor([-3], dtype=torch.int32, device=cuda)))
    assert torch.equal(dk.cpu(), k)


def test_recorded(cuda):
    """A fork, its copies and a compaction recorded once and replayed between eager steps."""
    S, P, left, chunk, D = 12, 16, 70, 2, 64
    dev, model = DevicePagePool(S, P, left, chunk, cuda), RaggedPool(S, P, left, chunk, range(S * 6))
    k = torch.randn(2, dev.num_pages, P, D, device=cuda)
    v = torch.randn_like(k)
    src, dst = _up([1, 1, 7], cuda), _up([3, 4, 0], cuda)

    def work():
        a = ops.page_fork(dev.state, src, dst)
        ops.kv_move_pages(k, v, a)
        b = ops.page_compact(dev.state)
        ops.kv_move_pages(k, v, b)
        return a, b

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.graph(graph, stream=side):
        a, b = work()
    torch.cuda.current_stream(cuda).wait_stream(side)
    _same(dev, model)  # recording ran nothing
    rng = np.random.default_rng(0)
    for turn in range(5):
        for _ in range(20):
            batch = rng.permutation(S)[: rng.integers(1, S + 1)]
            lengths = rng.integers(0, chunk + 1, len(batch))
            dev.advance(_up(batch, cuda), _up(lengths, cuda))
            model.advance(batch.tolist(), lengths.tolist())
        want = k.cpu()
        graph.replay()
        torch.cuda.synchronize()
        first, second = fork(model, [1, 1, 7], [3, 4, 0]), compact(model, dev.num_pages)
        assert _moves(a) == first and _moves(b) == second
        _same(dev, model)
        for f, t in first:
            want[:, t] = want[:, f]
        for f, t in second:
            want[:, t] = want[:, f]
        assert torch.equal(k.cpu(), want)


def test_encoder_streams_forked_and_compacted(cuda):
    """ModelCache: a forked row's windows and conv state are its source's and go on apart; compaction changes no window."""
    Ly, left, right, D, S = 3, 70, 1, 64, 6
    cache = ModelCache(Ly, (left, right), D, 9, batch_size=S, device=cuda, dtype=torch.float16, device_pages=True)
    plain = ModelCache(Ly, (left, right), D, 9, batch_size=S, device=cuda, dtype=torch.float16)
    g = torch.Generator(device=cuda).manual_seed(0)

    def step(dense):
        for layer in range(Ly):
            x = torch.randn(S, 2, D, generator=g, device=cuda).half()
            a = cache.update_attn_cache(layer, x, -x)
            b = plain.update_attn_cache(layer, x, -x)
            for got, want, old in zip(a, b, dense[layer]):
                # rows that were forked differ from the plain cache's where their window is older than the fork
                keep = torch.cat([old[:, 2:], want[:, -2:]], 1)
                assert torch.equal(got, keep)
            dense[layer] = [t.clone() for t in a]

    dense = [[torch.zeros(S, left + 2, D, device=cuda).half() for _ in range(2)] for _ in range(Ly)]
    for _ in range(45):
        step(dense)
    cache.conv_frames.normal_(generator=g)
    conv = cache.conv_frames.clone()
    cache.fork([4, 4, 0], [1, 5, 2])
    with pytest.raises(RuntimeError, match="moved"):
        cache.window(0)
    for layer in dense:
        for t in layer:
            t[[1, 5, 2]] = t[[4, 4, 0]]
    conv[[1, 5, 2]] = conv[[4, 4, 0]]
    assert torch.equal(cache.conv_frames, conv)
    for turn in range(30):
        step(dense)
        if turn % 7 == 3:
            cache.reset_slot(3)
            for layer in dense:
                for t in layer:
                    t[3] = 0
            cache.compact()
            assert sorted(cache.pool.free_list().tolist()) == cache.pool.free_list().tolist()


def test_rows_of_a_view_are_forked(cuda):
    """A view's rows name its own slots; a view whose step was open before the fork says so."""
    Ly, D, S = 2, 64, 5
    cache = ModelCache(Ly, (40, 1), D, 9, batch_size=S, device=cuda, dtype=torch.float16, device_pages=True)
    other = cache.batch([0, 2])
    g = torch.Generator(device=cuda).manual_seed(1)

    def step(view, n):
        return [view.update_attn_cache(layer, *(torch.randn(n, 2, D, generator=g, device=cuda).half() for _ in range(2))) for layer in range(Ly)]

    for _ in range(30):
        held = step(cache, S)
    cache.conv_frames.normal_(generator=g)
    view = cache.batch([3, 1, 4])
    step(other, 2)
    before = cache.conv_frames.clone()
    view.fork([0], [2])  # slot 3 into slot 4
    assert torch.equal(cache.conv_frames[4], before[3]) and torch.equal(cache.conv_frames[:4], before[:4])
    with pytest.raises(RuntimeError, match="moved"):
        other.window(0)
    after = step(cache, S)
    for old, new in zip(held, after):
        for a, b in zip(old, new):
            assert torch.equal(b[4, :-2], a[3, 2:]) and torch.equal(b[1, :-2], a[1, 2:]) and torch.equal(b[3, :-2], a[3, 2:])
    with pytest.raises(ValueError, match="rows"):
        view.fork([3], [0])
    with pytest.raises(ValueError, match="both"):
        view.fork([0, 1], [1, 2])
    with pytest.raises(ValueError, match="distinct"):
        view.fork([0, 0], [1, 1])
    assert torch.equal(cache.conv_frames[4], before[3])  # refused calls change nothing


def test_moves_of_a_cache_are_not_recorded(cuda):
    """A cache counts its moves on the host: neither a fork nor a compaction goes into a graph."""
    cache = ModelCache(1, (20, 1), 64, 9, batch_size=3, device=cuda, dtype=torch.float16, device_pages=True)
    x = torch.randn(3, 2, 64, device=cuda).half()
    cache.update_attn_cache(0, x, x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x + 1  # a graph holds something
        for call in (lambda: cache.fork([0], [1]), cache.compact):
            with pytest.raises(RuntimeError, match="not recorded"):
                call()
    cache.window(0)  # not stale
