"""A pool's own window as the default of a chunk's attention, against the definition in 64 bits."""

import numpy as np
import pytest
import torch

from parakeet_amd import ops
from parakeet_amd.pool import DevicePagePool
from tests._attend_model import attend

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


class _Texts:
    """A pool's streams whose keys and values the host keeps whole."""

    def __init__(self, cuda, dtype, slots, P, left, chunk, heads, kv_heads, hd, seed):
        self.cuda, self.dtype, self.heads, self.kv_heads, self.hd = cuda, dtype, heads, kv_heads, hd
        self.rng, self.g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        self.pool = DevicePagePool(slots, P, left, chunk, cuda)
        shape = (1, self.pool.num_pages, P, kv_heads * hd)
        self.k_pool, self.v_pool = (torch.zeros(shape, dtype=dtype, device=cuda) for _ in range(2))
        self.held = [[torch.zeros(0, kv_heads * hd, dtype=dtype) for _ in range(2)] for _ in range(slots)]

    def step(self, T, lengths):
        """T tokens at most a stream, with the default window; the outputs are checked against the pool's left."""
        n, D, hd = len(lengths), self.kv_heads * self.hd, self.hd
        up = lambda a: torch.as_tensor(a, dtype=torch.int32).to(self.cuda)  # noqa: E731
        rows, place = self.pool.advance(up(np.arange(n)), up(lengths))
        pages = ops.PagedKV(self.k_pool, self.v_pool, rows, self.pool.max_pages, left=self.pool.left)
        k, v, q = (torch.randn(n, T, w, generator=self.g).to(self.dtype) for w in (D, D, self.heads * hd))
        ops.kv_append_slots(pages, 0, k.to(self.cuda), v.to(self.cuda), place[:, :T].contiguous())
        out = ops.chunk_attn(q.to(self.cuda), pages, 0, num_heads=self.heads, lengths=up(lengths)).cpu()
        for b, m in enumerate(lengths):
            A = len(self.held[b][0])
            self.held[b] = [torch.cat([old, new[b, :m]]) for old, new in zip(self.held[b], (k, v))]
            assert (out[b, m:] == 0).all()
            if m == 0:
                continue
            first = max(0, A - self.pool.left)
            i, j = A + torch.arange(m)[:, None], torch.arange(first, A + m)[None, :]
            seen = (j <= i) & (j >= i - self.pool.left)
            ks, vs = (x[first:].double() for x in self.held[b])
            for h in range(self.heads):
                c, kc = slice(h * hd, (h + 1) * hd), h // (self.heads // self.kv_heads) * hd
                want, tol = attend(q[b, :m, c].double(), ks[:, kc : kc + hd], vs[:, kc : kc + hd], seen, hd**-0.5, self.dtype)
                far = (out[b, :m, c].double() - want).abs()
                assert (far <= tol).all(), f"stream {b} at {A}, {m} of {T} tokens: {(far / tol).max():.2f} times the tolerance"


@pytest.mark.parametrize("dtype,P,left,chunk", [(F16, 16, 70, 40), (BF16, 16, 500, 64), (F32, 8, 33, 5), (BF16, 64, 20, 50), (F16, 4, 60, 36)])
def test_the_pools_window_is_the_default(cuda, dtype, P, left, chunk):
    """Ragged steps of a sliding pool, whole chunks, parts of them and single tokens in turn: without `left` each token
    sees the pool's `left` positions before it, wherever in a page it is and however many tokens come with it."""
    texts = _Texts(cuda, dtype, 3, P, left, chunk, 2, 1, 64, seed=P + left)
    for turn in range(24):
        print(f"[default] {dtype} P {P} turn {turn}", flush=True)
        T = (chunk, 1, int(texts.rng.integers(1, chunk + 1)))[turn % 3]
        texts.step(T, [T, *texts.rng.integers(0, T + 1, 2).tolist()])


def test_the_default_at_every_place_in_a_page(cuda):
    """Single tokens one after another past two rounds of the ring, beside a pool that takes them in chunks."""
    one, many = (_Texts(cuda, BF16, 1, 16, 50, 34, 1, 1, 64, seed=5) for _ in range(2))
    for _ in range(170):
        one.step(1, [1])
    for _ in range(5):
        many.step(34, [34])


@pytest.mark.parametrize("T", [1, 40])
def test_no_window(cuda, T):
    """Rows of no known window: refused without `left`, unless no other window fits the ring."""
    pool = torch.zeros(1, 8, 16, 64, dtype=F16, device=cuda)
    rows = torch.zeros(1, 9, dtype=torch.int32, device=cuda)
    q = torch.zeros(1, T, 64, dtype=F16, device=cuda)
    with pytest.raises(ValueError, match="left"):
        ops.chunk_attn(q, ops.PagedKV(pool, pool, rows, 8), 0, num_heads=1)
    with pytest.raises(ValueError, match="left is 200"):
        ops.chunk_attn(q, ops.PagedKV(pool, pool, rows, 8, left=200), 0, num_heads=1)
    ops.chunk_attn(q, ops.PagedKV(pool, pool, rows, 8, left=200), 0, num_heads=1, left=20)
    tight = ops.PagedKV(pool, pool, rows, (T + 14) // 16 + 1)
    fits = (tight.max_pages - 1) * 16 + 1 - T
    if fits == 0:
        ops.chunk_attn(q, tight, 0, num_heads=1)
    else:
        with pytest.raises(ValueError, match="left"):
            ops.chunk_attn(q, tight, 0, num_heads=1)
