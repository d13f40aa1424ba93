"""Windows some of whose pages are absent (ring entries outside the pool), against the definition in 64 bits over
the positions that are there."""

import numpy as np
import pytest
import torch

from parakeet_amd import ops
from tests._attend_model import attend, fill_pages

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# which of the n pages of a window are absent
GONE = {
    "none": lambda n: [],
    "first": lambda n: [0],
    "middle": lambda n: [n // 2],
    "last": lambda n: [n - 1],
    "every second": lambda n: range(1, n, 2),
    "all but one": lambda n: [i for i in range(n) if i != n // 3],
    "all": lambda n: range(n),
}


def _absent(cuda, dtype, hd, heads, kv_heads, P, T, left, A, gone, seed=0):
    """(out, query, pages, what each stream's tokens see, k, v, first positions)"""
    rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    n, M = len(A), (left + T + P - 2) // P + 2
    rows = np.full((n, 1 + M), -1, dtype=np.int32)
    rows[:, 0] = A
    rows[:, 1:] = rng.permutation(n * M).reshape(n, M)
    first, end = [max(0, a - left) for a in A], [a + T for a in A]
    kp, vp, k, v = fill_pages(rows, P, M, kv_heads * hd, first, end, dtype, g)
    N, seen = kp.shape[1], []
    for b in range(n):
        lo, hi = first[b] // P, (end[b] - 1) // P
        away = [lo + i for i in GONE[gone[b]](hi - lo + 1)]
        for x, page in enumerate(away):
            rows[b, 1 + page % M] = (-1, N, 2**31 - 1, -(2**31))[x % 4]
        i, j = A[b] + torch.arange(T)[:, None], torch.arange(first[b], end[b])[None, :]
        there = ~torch.isin(j // P, torch.tensor(away, dtype=torch.int64))
        seen.append((j <= i) & (j >= i - left) & there)
    q = torch.randn(n, T, heads * hd, generator=g).to(dtype)
    pages = ops.PagedKV(kp.to(cuda), vp.to(cuda), torch.from_numpy(rows).to(cuda), M)
    print(f"[absent] {dtype} hd {hd} heads {heads}/{kv_heads} P {P} T {T} left {left} A {A} {gone}", flush=True)
    out = ops.chunk_attn(q.to(cuda), pages, 1, num_heads=heads, left=left)
    torch.cuda.synchronize()
    return out.cpu(), q, pages, seen, k, v, first


def _check(out, q, seen, k, v, heads, kv_heads, hd, dtype, rows=None):
    for b in range(len(seen)):
        some = slice(None) if rows is None else rows[b]
        for h in range(heads):
            c, kc = slice(h * hd, (h + 1) * hd), h // (heads // kv_heads) * hd
            want, tol = attend(q[b, some, c].double(), k[b][:, kc : kc + hd].double(), v[b][:, kc : kc + hd].double(), seen[b][some], hd**-0.5, dtype)
            far = (out[b, some, c].double() - want).abs()
            assert (far <= tol).all(), f"stream {b} head {h}: {(far / tol).max():.2f} times the tolerance"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("P", [8, 16, 64])
@pytest.mark.parametrize("T", [1, 9, 33, 50, 300])
def test_absent_pages(cuda, dtype, P, T):
    """The first, a middle, the last page of a window, every second, all but one: few and many rows, rings
    that have gone round, 32 to 300 positions before."""
    gone = list(GONE)
    left = 300 if T < 300 else 32
    out, q, pages, seen, k, v, _ = _absent(cuda, dtype, 64, 2, 1, P, T, left, [299, 1000, 77, 2111, 640, 0, 5000], gone, seed=T + P)
    _check(out, q, seen, k, v, 2, 1, 64, dtype)
    out, q, pages, seen, k, v, _ = _absent(cuda, dtype, 128, 3, 3, P, T, 130, [1000, 500], ["middle", "every second"], seed=T)
    _check(out, q, seen, k, v, 3, 3, 128, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [1, 40, 130])
def test_absent_pages_of_a_split_axis(cuda, dtype, T):
    """Long windows, whose keys are shared out over workgroups: parts with and without absent pages, parts without any page."""
    for gone in ("middle", "every second", "last", "all but one"):
        out, q, pages, seen, k, v, _ = _absent(cuda, dtype, 64, 2, 2, 16, T, 4000, [9000], [gone], seed=T)
        _check(out, q, seen, k, v, 2, 2, 64, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [40, 90])
def test_rows_made_again(cuda, dtype, T):
    """Beside an absent page a value that is not finite, which some tokens of the chunk do not see: those are as the
    definition over the pages that are there."""
    A, left, P, hd, heads = 1000, 60, 16, 64, 2
    _, q, pages, seen, k, v, first = _absent(cuda, dtype, hd, heads, 1, P, T, left, [A], ["middle"])
    rows, M = pages.rows.cpu(), pages.max_pages
    at = A + 20
    if int(rows[0, 1 + at // P % M]) not in range(pages.k_pool.shape[1]):
        at += P
    ops.page_blocks(pages.v_pool)[1, int(rows[0, 1 + at // P % M]), :, at % P] = float("inf")
    out = ops.chunk_attn(q.to(cuda), pages, 1, num_heads=heads, left=left).cpu()
    sees = seen[0][:, at - first[0]]
    assert sees.any() and not sees.all()
    assert not torch.isfinite(out[0, sees]).any()
    v[0][at - first[0]] = 0  # of no row that is compared
    _check(out, q, seen, k, v, heads, 1, hd, dtype, rows=[~sees])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("gone", ["middle", "last"])
def test_absent_pages_far_into_a_whole_window(cuda, dtype, gone):
    """A window of hundreds of pages that one workgroup takes whole, since there are many streams (all on the same pages)."""
    T, hd = 40, 64
    _, q, pages, seen, k, v, _ = _absent(cuda, dtype, hd, 1, 1, 16, T, 9000, [20000], [gone])
    n = 192
    many = torch.randn(n, T, hd, generator=torch.Generator().manual_seed(1)).to(dtype)
    many[-1] = q[0]
    there = ops.PagedKV(pages.k_pool, pages.v_pool, pages.rows.repeat(n, 1), pages.max_pages)
    out = ops.chunk_attn(many.to(cuda), there, 1, num_heads=1, left=9000).cpu()
    for b in (0, 77, n - 1):
        _check(out[b : b + 1], many[b : b + 1], seen, k, v, 1, 1, hd, dtype)
