"""A text decoder's operators as they are used together: steps of streams that come, fork, end
and are compacted, eager and recorded; caches past 4 GB."""

import numpy as np
import pytest
import torch

from parakeet_amd import ops
from parakeet_amd.pool import DevicePagePool
from tests._attend_model import HALF, attend, norm_rotate, pool_places

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _up(a, cuda):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(cuda)


class _Streams:
    """A pool of `slots` streams, their pages in two layers, and what their pages should hold."""

    def __init__(self, cuda, dtype, slots, P, left, chunk, heads, kv_heads, hd, states, seed):
        self.cuda, self.dtype, self.P, self.left, self.chunk, self.heads, self.kv_heads, self.hd = cuda, dtype, P, left, chunk, heads, kv_heads, hd
        self.rng, self.g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        self.pool = DevicePagePool(slots, P, left, chunk, cuda)
        shape = (2, self.pool.num_pages, P, kv_heads * hd)
        self.k_pool, self.v_pool = (torch.full(shape, float("nan"), dtype=dtype, device=cuda) for _ in range(2))
        self.place = pool_places(self.k_pool)
        self.q_weight, self.k_weight = (self._randn(hd, scale=0.2, shift=1.0) for _ in range(2))
        self.inv = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
        self.held = [[[], []] for _ in range(slots)]  # of a slot and layer: (k, v) rows as the pages have them
        self.states = self._randn(slots, states, 2 * kv_heads * hd)
        self.state_lens = self.rng.integers(0, states + 1, slots)

    def _randn(self, *shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=self.g) * scale + shift).to(self.dtype)

    def step(self, slots, lengths):
        cuda, D, W, hd = self.cuda, self.kv_heads * self.hd, self.heads * self.hd, self.hd
        rows, place = self.pool.advance(_up(slots, cuda), _up(lengths, cuda))
        pages = ops.PagedKV(self.k_pool, self.v_pool, rows, self.pool.max_pages)
        A, at = rows[:, 0].cpu(), place.cpu()
        for layer in range(2):
            x = self._randn(len(slots), self.chunk, W + 2 * D)
            d = x.to(cuda)
            q = ops.qk_norm_append(d[..., :W], d[..., W : W + D], d[..., W + D :], pages, layer, place, num_heads=self.heads,
                                   q_weight=self.q_weight.to(cuda), k_weight=self.k_weight.to(cuda), inv_freq=self.inv.to(cuda))
            out = ops.chunk_attn(q, pages, layer, num_heads=self.heads, lengths=_up(lengths, cuda), left=self.left)
            enc = self.states[slots].to(cuda)
            lens = _up(self.state_lens[slots], cuda)
            cross = ops.cross_attn(q, enc[..., :D], enc[..., D:], num_heads=self.heads, lengths=lens)
            self._check(layer, slots, lengths, A, at, x, q.cpu(), out.cpu(), cross.cpu())

    def _check(self, layer, slots, lengths, A, at, x, q, out, cross):
        D, W, hd, T = self.kv_heads * self.hd, self.heads * self.hd, self.hd, self.chunk
        kp, vp = self.k_pool[layer].cpu().reshape(-1), self.v_pool[layer].cpu().reshape(-1)
        place = self.place[0]
        pos = A[:, None] + torch.arange(T)
        wk, size = norm_rotate(x[..., W : W + D].double().unflatten(-1, (-1, hd)), self.k_weight.double(), pos, self.inv, 1e-6, False)
        for b, (s, n) in enumerate(zip(slots.tolist(), lengths.tolist())):
            cells = place[at[b, :n].long() // self.P, at[b, :n].long() % self.P]
            k, v = kp[cells], vp[cells]
            tol = HALF[self.dtype] * wk[b, :n].abs() + 2.0**-19 * size[b, :n] + 2.0**-25
            assert ((k.double() - wk[b, :n].flatten(-2)).abs() <= tol.flatten(-2)).all(), "keys"
            assert torch.equal(v, x[b, :n, W + D :]), "values"
            self.held[s][layer] += list(zip(k, v))
            assert len(self.held[s][layer]) == A[b] + n
            assert (out[b, n:] == 0).all()
            first = max(0, int(A[b]) - self.left)
            for what, got, m, ks, vs, seen in (
                ("tokens", out[b], n, *self._past(s, layer, first), self._causal(int(A[b]), n, first)),
                ("states", cross[b], T, self.states[s, : self.state_lens[s], :D], self.states[s, : self.state_lens[s], D:],
                 torch.ones(T, int(self.state_lens[s]), dtype=torch.bool)),
            ):
                if m == 0 or len(ks) == 0:
                    assert (got == 0).all()
                    continue
                for h in range(self.heads):
                    c, kc = slice(h * hd, (h + 1) * hd), h // (self.heads // self.kv_heads) * hd
                    want, tol = attend(q[b, :m, c].double(), ks[:, kc : kc + hd].double(), vs[:, kc : kc + hd].double(), seen, hd**-0.5, self.dtype)
                    far = (got[:m, c].double() - want).abs()
                    assert (far <= tol).all(), f"{what}: stream {b} slot {s} head {h}: {(far / tol).max():.2f} times the tolerance"

    def _past(self, s, layer, first):
        rows = self.held[s][layer][first:]
        return (torch.stack([r[i] for r in rows]) if rows else torch.zeros(0, self.kv_heads * self.hd, dtype=self.dtype) for i in (0, 1))

    def _causal(self, A, n, first):
        i, j = A + torch.arange(n)[:, None], torch.arange(first, A + n)[None, :]
        return (j <= i) & (j >= i - self.left)

    def fork(self, src, dst):
        ops.kv_move_pages(self.k_pool, self.v_pool, self.pool.fork(src, dst))
        for s, d in zip(src, dst):
            self.held[d] = [list(x) for x in self.held[s]]

    def end(self, gone):
        self.pool.reset_slots(gone)
        for s in gone:
            self.held[s] = [[], []]

    def compact(self):
        ops.kv_move_pages(self.k_pool, self.v_pool, self.pool.compact())
        # what no slot holds from here on is never read again
        held = self.pool.state.ring[self.pool.state.ring >= 0].long()
        free = torch.ones(self.pool.num_pages, dtype=torch.bool, device=self.cuda)
        free[held] = False
        for pool in (self.k_pool, self.v_pool):
            pool[:, free] = float("nan")


@pytest.mark.parametrize("dtype,slots,P,left,chunk,heads,kv_heads,hd", [(BF16, 7, 16, 90, 5, 4, 2, 64), (F16, 6, 8, 40, 1, 2, 2, 128), (F32, 5, 16, 33, 4, 3, 1, 64),
                                                                    (F16, 4, 4, 300, 40, 4, 1, 64)])
def test_streams_come_fork_and_end(cuda, dtype, slots, P, left, chunk, heads, kv_heads, hd):
    st = _Streams(cuda, dtype, slots, P, left, chunk, heads, kv_heads, hd, 37, seed=slots)
    for turn in range(18):
        print(f"[decoder] {dtype} turn {turn}", flush=True)
        batch = st.rng.permutation(slots)[: st.rng.integers(1, slots + 1)]
        st.step(batch, st.rng.integers(0, chunk + 1, len(batch)))
        if turn % 4 == 1:
            both = st.rng.permutation(slots)
            st.fork(st.rng.choice(both[2:], 2).tolist(), both[:2].tolist())
        if turn % 5 == 3:
            st.end([int(st.rng.integers(0, slots))])
            st.compact()


@pytest.mark.parametrize("dtype,T,left", [(BF16, 1, 3000), (F16, 5, 200), (BF16, 70, 400), (F32, 3, 100)])
def test_a_recorded_step(cuda, dtype, T, left):
    """A step of all four launches recorded once and replayed with new tokens, eager work between: every replay has
    the bits of the eager step on a pool of its own."""
    B, P, heads, kv, hd, S = 5, 16, 8, 2, 64, 200
    W, D = heads * hd, kv * hd
    g = torch.Generator(device=cuda).manual_seed(3)
    pools = [DevicePagePool(B, P, left, T, cuda) for _ in range(2)]
    kv_of = [[torch.zeros(1, pools[0].num_pages, P, D, dtype=dtype, device=cuda) for _ in range(2)] for _ in range(2)]
    x = torch.zeros(B, T, W + 2 * D, dtype=dtype, device=cuda)
    lengths = torch.full((B,), T, dtype=torch.int32, device=cuda)
    slots = torch.arange(B, dtype=torch.int32, device=cuda)
    enc = torch.randn(B, S, 2 * D, generator=g, device=cuda).to(dtype)
    lens = torch.tensor([S, 0, 1, 77, S], dtype=torch.int32, device=cuda)
    w = torch.ones(hd, dtype=dtype, device=cuda)
    inv = (10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)).to(cuda)

    def step(i):
        rows, place = ops.page_step(pools[i].state, slots, lengths)
        pages = ops.PagedKV(*kv_of[i], rows, pools[i].max_pages)
        q = ops.qk_norm_append(x[..., :W], x[..., W : W + D], x[..., W + D :], pages, 0, place, num_heads=heads, q_weight=w, k_weight=w, inv_freq=inv)
        a = ops.chunk_attn(q, pages, 0, num_heads=heads, lengths=lengths, left=left)
        return a, ops.cross_attn(a, enc[..., :D], enc[..., D:], num_heads=heads, lengths=lens)

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.graph(graph, stream=side):
        out = step(0)
    torch.cuda.current_stream(cuda).wait_stream(side)
    for turn in range(8 if left < 1000 else 40):
        x.copy_(torch.randn(x.shape, generator=g, device=cuda).to(dtype))
        lengths.copy_(torch.randint(0, T + 1, (B,), generator=g, device=cuda))
        want = [t.clone() for t in step(1)]
        _ = torch.randn(512, 512, device=cuda) @ torch.randn(512, 512, device=cuda)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), f"replay {turn}"
        for a, b in zip(kv_of[0], kv_of[1]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 50])
def test_pages_past_4_gb(cuda, T):
    """A layer's slab of 5 GB whose last pages, and its first, are a stream's: written and read at their places."""
    P, heads, hd, left = 16, 2, 128, 100
    D, M = hd, (left + T + P - 2) // P + 1
    N = 5 * 2**30 // (P * D * 2)
    kp, vp = (torch.empty(1, N, P, D, dtype=BF16, device=cuda) for _ in range(2))
    pages = list(range(N - M + 1, N)) + [0]
    rows = torch.tensor([[left] + pages], dtype=torch.int32, device=cuda)
    g = torch.Generator().manual_seed(0)
    n = left + T
    x = torch.randn(1, n, (heads + 2) * hd, generator=g).to(BF16)
    slot = torch.tensor([[pages[p // P % M] * P + p % P for p in range(n)]], dtype=torch.int32)
    assert int(slot.max()) * D * 2 > 2**32
    d = x.to(cuda)
    paged = ops.PagedKV(kp, vp, rows, M)
    q = ops.qk_norm_append(d[..., : 2 * hd], d[..., 2 * hd : 3 * hd], d[..., 3 * hd :], paged, 0, slot.to(cuda), num_heads=heads)
    assert torch.equal(q, d[..., : 2 * hd])
    blocks = ops.page_blocks(vp)[0]
    at = slot[0].long().to(cuda)
    assert torch.equal(blocks[at // P, :, at % P].reshape(n, D), d[0, :, 3 * hd :])
    out = ops.chunk_attn(q[:, left:], paged, 0, num_heads=heads, left=left)
    seen = torch.arange(n)[None, :] <= left + torch.arange(T)[:, None]
    seen &= torch.arange(n)[None, :] >= torch.arange(T)[:, None]
    for h in range(heads):
        c = slice(h * hd, (h + 1) * hd)
        want, tol = attend(x[0, left:, c].double(), x[0, :, 2 * hd : 3 * hd].double(), x[0, :, 3 * hd :].double(), seen, hd**-0.5, BF16)
        assert ((out[0, :, c].double().cpu() - want).abs() <= tol).all()
    moved = ops.PageMoves(torch.tensor([[N - 1, 1]], dtype=torch.int32, device=cuda), torch.ones(1, dtype=torch.int32, device=cuda))
    ops.kv_move_pages(kp, vp, moved)
    assert torch.equal(kp[0, 1], kp[0, N - 1]) and torch.equal(vp[0, 1], vp[0, N - 1])


@pytest.mark.parametrize("T", [2, 60])
def test_states_past_4_gb(cuda, T):
    """Streams 3 GB and states 1 MB apart in memory."""
    hd, S, B = 64, 2500, 2
    st, sb = 2**19, 3 * 2**29
    memory = torch.empty(sb + S * st, dtype=F16, device=cuda)
    kv = memory.as_strided((B, S, 2 * hd), (sb, st, 1))
    g = torch.Generator().manual_seed(0)
    x = torch.randn(B, S, 2 * hd, generator=g).to(F16)
    kv.copy_(x.to(cuda))
    q = torch.randn(B, T, hd, generator=g).to(F16)
    out = ops.cross_attn(q.to(cuda), kv[..., :hd], kv[..., hd:], num_heads=1).cpu()
    for b in range(B):
        want, tol = attend(q[b].double(), x[b, :, :hd].double(), x[b, :, hd:].double(), torch.ones(T, S, dtype=torch.bool), hd**-0.5, F16)
        assert ((out[b].double() - want).abs() <= tol).all()
