"""New tokens over a paged cache and over the encoder's states, against the definition in
64 bits, at every kind of size: what no query sees is NaN in every test's memory."""

import math

import numpy as np
import pytest
import torch

from parakeet_amd import ops
from tests._attend_model import attend, fill_pages

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rows(A, new, left, T, P, M, rng):
    """Block-table rows of streams that hold the pages of their windows, pages in no order."""
    n = len(A)
    pages = rng.permutation(n * M).reshape(n, M)
    rows = np.full((n, 1 + M), -1, dtype=np.int32)
    rows[:, 0] = A
    for b in range(n):
        end = A[b] + new[b]
        for k in range(max(0, end - left - T) // P, (end + P - 1) // P):
            rows[b, 1 + k % M] = pages[b, k % M]
    return rows


def _check(out, want, tol, what):
    out, far = out.double().cpu(), (out.double().cpu() - want).abs()
    assert torch.isfinite(out).all(), f"{what}: not finite"
    worst = (far / tol).max().item() if far.numel() else 0.0
    assert worst <= 1, f"{what}: {worst:.2f} times the tolerance"


def _chunk(cuda, dtype, hd, heads, kv_heads, P, T, left, A, new, seed=0, whole=None, scale=None, extra_ring=0):
    rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    M = (left + T + P - 2) // P + 1 + extra_ring
    n, D = len(A), kv_heads * hd
    rows = _rows(A, new, left, T, P, M, rng)
    first = [max(0, a - left) for a in A]
    end = [a + m for a, m in zip(A, new)]
    end = [e if m else f for e, f, m in zip(end, first, new)]
    kp, vp, k, v = fill_pages(rows, P, M, D, first, end, dtype, g)
    q = torch.randn(n, T, heads * hd, generator=g).to(dtype)
    lengths = None if whole else torch.tensor(new, dtype=torch.int32, device=cuda)
    pages = ops.PagedKV(kp.to(cuda), vp.to(cuda), torch.from_numpy(rows).to(cuda), M)
    print(f"[chunk] {dtype} hd {hd} heads {heads}/{kv_heads} P {P} T {T} left {left} A {A} new {new}", flush=True)
    out = ops.chunk_attn(q.to(cuda), pages, 1, num_heads=heads, lengths=lengths, left=left, scale=scale)
    torch.cuda.synchronize()
    s = scale or hd**-0.5
    for b in range(n):
        i = torch.arange(new[b])[:, None] + A[b]
        j = torch.arange(first[b], end[b])[None, :]
        seen = (j <= i) & (j >= i - left)
        assert (out[b, new[b] :] == 0).all(), "tokens past a stream's"
        for h in range(heads):
            c = slice(h * hd, (h + 1) * hd)
            kc = slice(h // (heads // kv_heads) * hd, (h // (heads // kv_heads) + 1) * hd)
            if new[b] == 0:
                continue
            want, tol = attend(q[b, : new[b], c].double(), k[b][:, kc].double(), v[b][:, kc].double(), seen, s, dtype)
            _check(out[b, : new[b], c], want, tol, f"stream {b} head {h}")
    return out, q, pages


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd,heads,kv_heads", [(64, 8, 8), (64, 6, 2), (128, 8, 1), (128, 2, 2), (64, 5, 1), (128, 32, 2)])
def test_single_tokens(cuda, dtype, hd, heads, kv_heads):
    """One new token over caches from empty to hundreds, odd lengths, pages ending inside tiles."""
    A = [0, 1, 15, 16, 17, 63, 64, 100, 511, 300]
    _chunk(cuda, dtype, hd, heads, kv_heads, 16, 1, 511, A, [1] * len(A))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("P", [1, 2, 4, 8, 32, 64, 256])
def test_page_sizes(cuda, dtype, P):
    _chunk(cuda, dtype, 64, 4, 2, P, 3, 150, [0, 5, 149, 150, 333], [3, 2, 3, 1, 3])
    _chunk(cuda, dtype, 128, 4, 2, P, 40, 150, [0, 149, 333], [40, 33, 1])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [2, 5, 7, 16, 17, 31, 33, 64, 65, 130, 257])
def test_chunks(cuda, dtype, T):
    """Tokens of a chunk, whole and ragged streams, one without tokens, before and behind a window."""
    _chunk(cuda, dtype, 64, 4, 2, 16, T, 97, [0, 40, 97, 400, 33], [T, T, max(1, T - 1), T // 2, 0])
    _chunk(cuda, dtype, 128, 3, 1, 16, T, 3, [0, 1, 200], [T, 1, T])
    _chunk(cuda, dtype, 64, 2, 2, 8, T, 0, [0, 7], [T, T])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,heads,kv_heads,T,A", [(128, 8, 2, 300, [1000, 17]), (64, 16, 1, 64, [2111]), (128, 16, 16, 128, [700])])
def test_many_rows(cuda, dtype, hd, heads, kv_heads, T, A):
    _chunk(cuda, dtype, hd, heads, kv_heads, 32, T, 2200, A, [T] * len(A), whole=True)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_long_cache(cuda, dtype):
    """One token far into a long cache: the axis is split over workgroups and joined."""
    _chunk(cuda, dtype, 64, 2, 1, 16, 1, 20000, [19999, 5], [1, 1])
    _chunk(cuda, dtype, 128, 8, 1, 16, 3, 9000, [8990], [3])


@pytest.mark.parametrize("dtype,n,heads,kv_heads,T", [(BF16, 70, 8, 4, 1), (F16, 70, 2, 2, 2), (BF16, 17, 8, 8, 1), (F32, 64, 5, 5, 1), (F16, 66, 4, 4, 33)])
def test_many_streams_over_caches_of_any_lengths(cuda, dtype, n, heads, kv_heads, T):
    rng = np.random.default_rng(n)
    A, new = rng.integers(0, 2500, n), rng.integers(0, T + 1, n)
    A[1], A[2], new[2], new[3] = 0, A[4], T, 0
    _chunk(cuda, dtype, 64, heads, kv_heads, 16, T, 1100, A.tolist(), new.tolist())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [1, 6, 40])
def test_far_positions(cuda, dtype, T):
    """Rings that have gone round, up to the last positions that a row can hold."""
    top = 2**31 - 1 - T
    _chunk(cuda, dtype, 64, 2, 1, 16, T, 77, [top, top - 5, 10**9 + 7], [T, T, T], extra_ring=3)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_scale_and_large_scores(cuda, dtype):
    """Scores of hundreds: the running maximum moves by more than a type's range."""
    _chunk(cuda, dtype, 64, 2, 1, 16, 1, 300, [299], [1], scale=20.0)
    _chunk(cuda, dtype, 128, 2, 1, 16, 37, 300, [299], [37], scale=6.0)


@pytest.mark.parametrize("T", [1, 9, 50])
def test_absent_streams_and_counts_out_of_range(cuda, T):
    """Rows of -1 (an absent stream) give zeros; token counts are held within 0 .. T."""
    g = torch.Generator().manual_seed(1)
    M, P, D = 8, 16, 64
    rows = torch.full((3, 1 + M), -1, dtype=torch.int32)
    rows[:, 0] = torch.tensor([0, 50, 20])
    rows[2, 1:] = torch.arange(M)
    kp, vp = (torch.randn(1, M, P, D, generator=g).to(F16).to(cuda) for _ in range(2))
    q = torch.randn(3, T, D, generator=g).to(F16).to(cuda)
    pages = ops.PagedKV(kp, vp, rows.to(cuda), M)
    long = ops.chunk_attn(q, pages, 0, num_heads=1, lengths=torch.tensor([T, T, T + 9], dtype=torch.int32, device=cuda), left=60)
    whole = ops.chunk_attn(q, pages, 0, num_heads=1, left=60)
    assert (long[:2] == 0).all() and torch.equal(long, whole) and torch.isfinite(long).all() and (long[2] != 0).any()
    none = ops.chunk_attn(q, pages, 0, num_heads=1, lengths=torch.tensor([-4, 0, -1], dtype=torch.int32, device=cuda), left=60)
    assert (none == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("T", [4, 70])
def test_what_is_not_seen_is_not_felt(cuda, dtype, bad, T):
    """K and V of one token not finite: tokens before it, and those whose window has left it, are as
    without; the others are NaN where the definition is."""
    A, left, P, hd, at = 40, 30, 16, 64, 41
    out, q, pages = _chunk(cuda, dtype, hd, 2, 1, P, T, left, [A], [T])
    rows, M = pages.rows.cpu().numpy(), pages.max_pages
    page = int(rows[0, 1 + at // P % M])
    for pool in (pages.k_pool, pages.v_pool):
        ops.page_blocks(pool)[1, page, :, at % P] = bad
    again = ops.chunk_attn(q.to(cuda), pages, 1, num_heads=2, left=left, lengths=torch.tensor([T], dtype=torch.int32, device=cuda))
    i = torch.arange(T) + A
    sees = (i >= at) & (i - at <= left)
    assert torch.isfinite(again[0, ~sees]).all()
    # the rows that do not see it may be summed in another order
    assert torch.allclose(again[0, ~sees].double(), out[0, ~sees].double(), rtol=4 * torch.finfo(dtype).eps, atol=4 * torch.finfo(dtype).eps)
    assert not torch.isfinite(again[0, sees]).any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd,heads,T,n", [(64, 2, 4, 2), (64, 2, 70, 41), (128, 3, 50, 20), (128, 4, 40, 33)])
def test_tokens_past_a_stream_feel_nothing(cuda, dtype, hd, heads, T, n):
    """A value that is not finite, of a position that a stream's last tokens see: the tokens past them
    are zeros all the same."""
    A, left, P = 40, 200, 16
    at = A + n - 1
    out, q, pages = _chunk(cuda, dtype, hd, heads, 1, P, T, left, [A], [n])
    rows, M = pages.rows.cpu().numpy(), pages.max_pages
    ops.page_blocks(pages.v_pool)[1, int(rows[0, 1 + at // P % M]), :, at % P] = float("inf")
    again = ops.chunk_attn(q.to(cuda), pages, 1, num_heads=heads, left=left, lengths=torch.tensor([n], dtype=torch.int32, device=cuda))
    assert (again[0, n:] == 0).all()
    assert not torch.isfinite(again[0, n - 1]).any()
    assert torch.allclose(again[0, : n - 1].double(), out[0, : n - 1].double(), rtol=4 * torch.finfo(dtype).eps, atol=4 * torch.finfo(dtype).eps)


def test_layouts(cuda):
    """A query that is a view of a wider projection, rows of a wider block table, an output that is a
    view, the query itself as output: the same bits as the plain call."""
    out, q, pages = _chunk(cuda, BF16, 128, 4, 2, 16, 5, 100, [80, 3], [5, 4])
    lengths = torch.tensor([5, 4], dtype=torch.int32, device=cuda)
    wide = torch.full((2, 9, 3 * 512), float("nan"), dtype=BF16, device=cuda)
    wide[:, 2:7, 512:1024] = q.to(cuda)
    rows = torch.full((4, pages.rows.shape[1] + 6), 12345, dtype=torch.int32, device=cuda)
    rows[:2, : pages.rows.shape[1]] = pages.rows
    there = ops.PagedKV(pages.k_pool, pages.v_pool, rows, pages.max_pages)
    call = lambda query, **kw: ops.chunk_attn(query, there, 1, num_heads=4, lengths=lengths, left=100, **kw)  # noqa: E731
    assert torch.equal(call(wide[:, 2:7, 512:1024]), out)
    hold = torch.full((2, 6, 640), 7.0, dtype=BF16, device=cuda)
    assert torch.equal(call(wide[:, 2:7, 512:1024], out=hold[:, :5, 64:576]), out)
    assert (hold[:, 5] == 7).all() and (hold[..., :64] == 7).all() and (hold[..., 576:] == 7).all()
    own = q.to(cuda)
    assert call(own, out=own) is own and torch.equal(own, out)
    assert torch.equal(ops.chunk_attn(q.to(cuda)[:, :0], there, 1, num_heads=4), out[:, :0])
    assert ops.chunk_attn(q.to(cuda)[:0], there, 1, num_heads=4).shape == (0, 5, 512)


def test_a_query_of_all_streams(cuda):
    """One row of queries for all streams and all tokens (strides of 0): the bits of its copies."""
    _, _, pages = _chunk(cuda, BF16, 64, 4, 2, 16, 3, 100, [80, 3], [3, 3], whole=True)
    q = torch.randn(1, 1, 256, device=cuda).to(BF16)
    many = q.expand(2, 3, -1)
    got = ops.chunk_attn(many, pages, 1, num_heads=4, left=100)
    assert torch.equal(got, ops.chunk_attn(many.contiguous(), pages, 1, num_heads=4, left=100)) and torch.isfinite(got).all()
    kv = torch.randn(2, 70, 256, device=cuda).to(BF16)
    assert torch.equal(ops.cross_attn(many, kv, kv, num_heads=4), ops.cross_attn(many.contiguous(), kv, kv, num_heads=4))


def test_two_streams_at_once(cuda):
    """Split calls that run at the same time on two streams keep apart: the bits of one after another."""
    _, q, pages = _chunk(cuda, BF16, 128, 8, 2, 16, 1, 9000, [8999, 700, 5000], [1, 1, 1])
    q = [x.to(cuda) for x in (q, -q, q * 0.5, q * 0.25)]
    kv = torch.randn(3, 4000, 512, device=cuda).to(BF16)
    k, v = kv[..., :256], kv[..., 256:]
    calls = [lambda x: ops.chunk_attn(x, pages, 1, num_heads=8, left=9000), lambda x: ops.cross_attn(x, k, v, num_heads=8)]
    want = [call(x) for x in q for call in calls]
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for x in q:
        for call, stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                got.append(call(x))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_another_stream_and_repeats(cuda):
    """On a side stream, and twice: the same bits."""
    out, q, pages = _chunk(cuda, F16, 64, 8, 1, 16, 1, 9000, [8999, 100, 5000], [1, 1, 1])
    q, lengths = q.to(cuda), torch.tensor([1, 1, 1], dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        there = ops.chunk_attn(q, pages, 1, num_heads=8, lengths=lengths, left=9000)
    torch.cuda.current_stream(cuda).wait_stream(side)
    for _ in range(3):
        assert torch.equal(ops.chunk_attn(q, pages, 1, num_heads=8, lengths=lengths, left=9000), out)
    assert torch.equal(there, out)


# ---------------------------------------------------------------------------
# states


def _cross(cuda, dtype, hd, heads, kv_heads, T, S, lens, seed=0, expand=False, scale=None):
    g = torch.Generator().manual_seed(seed)
    n, D = len(lens), kv_heads * hd
    kv = torch.randn(1 if expand else n, S, 2 * D, generator=g).to(dtype)
    for b in range(kv.shape[0]):
        kv[b, max(lens) if expand else lens[b] :] = float("nan")
    q = torch.randn(n, T, heads * hd, generator=g).to(dtype)
    print(f"[cross] {dtype} hd {hd} heads {heads}/{kv_heads} T {T} S {S} lens {lens}", flush=True)
    dev = kv.to(cuda)
    k, v = (x.expand(n, -1, -1) for x in (dev[..., :D], dev[..., D:])) if expand else (dev[..., :D], dev[..., D:])
    out = ops.cross_attn(q.to(cuda), k, v, num_heads=heads, lengths=torch.tensor(lens, dtype=torch.int32, device=cuda), scale=scale)
    torch.cuda.synchronize()
    for b in range(n):
        if lens[b] == 0:
            assert (out[b] == 0).all()
            continue
        x = kv[0 if expand else b, : lens[b]].double()
        for h in range(heads):
            c, kh = slice(h * hd, (h + 1) * hd), h // (heads // kv_heads) * hd
            seen = torch.ones(T, lens[b], dtype=torch.bool)
            want, tol = attend(q[b, :, c].double(), x[:, kh : kh + hd], x[:, D + kh : D + kh + hd], seen, scale or hd**-0.5, dtype)
            _check(out[b, :, c], want, tol, f"stream {b} head {h}")
    return out, q, dev


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd,heads,kv_heads", [(64, 8, 8), (128, 6, 2), (64, 16, 1)])
@pytest.mark.parametrize("T", [1, 4, 21, 65])
def test_states(cuda, dtype, hd, heads, kv_heads, T):
    _cross(cuda, dtype, hd, heads, kv_heads, T, 131, [131, 0, 1, 17, 64, 130])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_states_shared_and_long(cuda, dtype):
    _cross(cuda, dtype, 64, 2, 1, 3, 700, [700, 650, 3], expand=True)
    _cross(cuda, dtype, 128, 2, 2, 1, 6001, [6001], scale=0.3)
    _cross(cuda, dtype, 64, 4, 4, 150, 333, [333, 7])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [1, 20, 140])
def test_a_state_for_all(cuda, dtype, T):
    """States that are one row (a stride of 0 along them): the mean of equal values is the value, up to
    the weights' and the quotient's roundings."""
    g = torch.Generator().manual_seed(3)
    q, kv = torch.randn(2, T, 128, generator=g).to(dtype), torch.randn(2, 1, 256, generator=g).to(dtype)
    k, v = (x.expand(-1, 90, -1) for x in (kv.to(cuda)[..., :128], kv.to(cuda)[..., 128:]))
    out = ops.cross_attn(q.to(cuda), k, v, num_heads=2, lengths=torch.tensor([90, 33], dtype=torch.int32, device=cuda))
    want = kv[..., 128:].double().expand(-1, T, -1)
    # output and weights each rounded once to the type; 2^-20: fp32 sums of 90 weights, exp2 and the quotient
    tol = (3 * torch.finfo(dtype).eps / 2 + 2.0**-20) * want.abs() + (2.0**-25 if dtype is F16 else 0)
    _check(out, want, tol, "one state")


@pytest.mark.parametrize("dtype,n,heads,kv_heads,T", [(F16, 40, 8, 8, 4), (BF16, 64, 8, 8, 1), (F16, 130, 4, 2, 3), (BF16, 70, 8, 8, 2), (F32, 45, 7, 7, 9),
                                                      (BF16, 20, 4, 4, 600), (F16, 30, 4, 4, 700), (F32, 9, 4, 4, 300), (BF16, 300, 2, 1, 2), (F16, 290, 2, 2, 1)])
def test_many_streams_of_any_lengths(cuda, dtype, n, heads, kv_heads, T):
    """Batches whose workgroups are more than the CUs: each stream is answered once, in whatever order they are taken."""
    rng, S = np.random.default_rng(n), 530
    lens = rng.integers(0, S + 1, n).tolist()
    lens[1], lens[2], lens[3], lens[n - 1], lens[n - 2] = 0, S, S, 1, lens[4]
    _cross(cuda, dtype, 64, heads, kv_heads, T, S, lens)


def test_no_states(cuda):
    q = torch.randn(2, 3, 128, device=cuda, dtype=F16)
    kv = torch.empty(2, 0, 128, device=cuda, dtype=F16)
    assert (ops.cross_attn(q, kv, kv, num_heads=2) == 0).all()
    kv = torch.empty(2, 5, 128, device=cuda, dtype=F16)
    assert ops.cross_attn(q[:, :0], kv, kv, num_heads=2).shape == (2, 0, 128)
    own = q.clone()
    lengths = torch.zeros(2, dtype=torch.int32, device=cuda)
    assert ops.cross_attn(own, kv, kv, num_heads=2, lengths=lengths, out=own) is own and (own == 0).all()


def test_autocast_to_another_type_is_refused(cuda):
    q = torch.randn(1, 2, 64, device=cuda)
    pool = torch.zeros(1, 1, 16, 64, device=cuda)
    pages = ops.PagedKV(pool, pool.clone(), torch.zeros(1, 2, dtype=torch.int32, device=cuda), 1)
    slots = torch.full((1, 2), -1, dtype=torch.int32, device=cuda)
    for call in (lambda: ops.cross_attn(q, q, q, num_heads=1), lambda: ops.chunk_attn(q[:, :1], pages, 0, num_heads=1),
                 lambda: ops.qk_norm_append(q, q, q, pages, 0, slots, num_heads=1)):
        with torch.autocast("cuda", dtype=torch.bfloat16), pytest.raises(RuntimeError, match="autocast"):
            call()
        with torch.autocast("cuda", dtype=torch.float32, enabled=False):
            call()


def test_outputs_that_meet_operands_are_refused(cuda):
    q = torch.randn(1, 4, 128, device=cuda, dtype=F16)
    kv = torch.randn(1, 9, 128, device=cuda, dtype=F16)
    pages = ops.PagedKV(kv[:, :8].reshape(1, 1, 8, 128), torch.zeros(1, 1, 8, 128, device=cuda, dtype=F16), torch.zeros(1, 2, dtype=torch.int32, device=cuda), 1)
    for out in (kv[:, :4], kv[:, 5:]):
        with pytest.raises(ValueError, match="overlap"):
            ops.cross_attn(q, kv, kv, num_heads=2, out=out)
    wide = torch.randn(1, 5, 128, device=cuda, dtype=F16)
    with pytest.raises(ValueError, match="overlap"):
        ops.cross_attn(wide[:, :4], kv, kv, num_heads=2, out=wide[:, 1:])
    with pytest.raises(ValueError, match="overlap"):
        ops.chunk_attn(q[:, :1], pages, 0, num_heads=2, out=pages.v_pool.view(1, 8, 128)[:, 3:4])
    with pytest.raises(ValueError, match="overlap"):
        ops.cross_attn(q.expand(2, -1, -1), kv.expand(2, -1, -1), kv.expand(2, -1, -1), num_heads=2, out=q.expand(2, -1, -1))


def test_outputs_that_something_follows_are_refused(cuda):
    q, kv = torch.randn(1, 2, 64, device=cuda), torch.randn(1, 9, 64, device=cuda)
    pool = torch.zeros(1, 1, 16, 64, device=cuda)
    pages = ops.PagedKV(pool, pool.clone(), torch.zeros(1, 3, dtype=torch.int32, device=cuda), 2)
    slots = torch.zeros(1, 2, dtype=torch.int32, device=cuda)
    weight = torch.ones(64, device=cuda)
    calls = [lambda out: ops.cross_attn(q, kv, kv, num_heads=1, out=out), lambda out: ops.chunk_attn(q, pages, 0, num_heads=1, left=4, out=out),
             lambda out: ops.qk_norm_append(q, kv[:, :2], kv[:, 2:4], pages, 0, slots, num_heads=1, q_weight=weight, out=out)]
    for call in calls:
        leaf = torch.zeros_like(q, requires_grad=True)
        with pytest.raises(RuntimeError, match="no backward"):
            call(leaf)
        with torch.no_grad():
            assert call(leaf) is leaf
    with pytest.raises(ValueError, match="overlap"):
        ops.qk_norm_append(q[:, :1], kv[:, :1], kv[:, 1:2], pages, 0, slots[:, :1], num_heads=1, q_weight=weight, out=weight.view(1, 1, 64))
