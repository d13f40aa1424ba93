"""Attention over scores at the ends of a type's range: one key far above a long tail of others, scores of -inf, scores
of which fp32 knows large steps only."""

import math

import pytest
import torch

from parakeet_amd import ops
from tests._attend_model import HALF, pool_places

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _paged(cuda, k, v, P, T):
    """One stream's keys and values [L, D], the last T of them a step's, on pages in reverse order."""
    L, D = k.shape
    n = (L + P - 1) // P
    pools = []
    for x in (k, v):
        pool = torch.full((1, n, P, D), float("nan"), dtype=x.dtype)
        pos = torch.arange(L)
        pool.view(-1)[pool_places(pool)[0, n - 1 - pos // P, pos % P]] = x
        pools.append(pool.to(cuda))
    rows = torch.tensor([[L - T] + list(range(n - 1, -1, -1)) + [-1] * (T // P + 2)], dtype=torch.int32, device=cuda)
    return ops.PagedKV(*pools, rows, rows.shape[1] - 1)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bits", [16.25, 20.5, 25.25])
@pytest.mark.parametrize("top", [0, 7777, 19999])
@pytest.mark.parametrize("T", [1, 40])
def test_a_long_tail(cuda, dtype, bits, top, T):
    """20,000 keys whose weights are 2^-bits of one key's, which is first, last or between, and whose value is 0:
    the output is the tail's mass times its values, for texts over states and tokens over pages.

    How far a kernel may be, with u half a step of the type and p the tail's mass (n 2^-bits / (1 + n 2^-bits)):
    the output's rounding, a weight's before the product with its value and its sum's, u each; fp32 sums over n
    keys in tiles of 16: 2^-24 a tile; a score of `bits` and its product with log2 e, each rounded, exp2 and the quotient: 2^-18."""
    n, hd, heads = 20000, 64, 2
    g = torch.Generator().manual_seed(top)
    # the key's score: q . k = (bits / log2 e) in its first column, in fp32; 16-bit types: the nearest they have
    high = torch.tensor(bits / math.log2(math.e)).to(dtype)
    weight = 2.0 ** (-float(high) * math.log2(math.e))
    q = torch.zeros(1, T, heads * hd).to(dtype)
    q[..., ::hd] = 1
    k = torch.zeros(n, heads * hd).to(dtype)
    k[top, ::hd] = high
    v = (torch.rand(n, heads * hd, generator=g) + 0.5).to(dtype)
    v[top] = 0
    u, total = HALF[dtype], 1 + (n - 1) * weight
    want = weight * v.double().sum(0) / total
    tol = (3 * u + 2.0**-18 + n / 16 * 2.0**-24) * want
    print(f"[tail] {dtype} bits {bits} top {top} T {T}", flush=True)
    kd, vd = (x[None].to(cuda) for x in (k, v))
    out = ops.cross_attn(q.to(cuda), kd, vd, num_heads=heads, scale=1.0).double().cpu()
    far = ((out - want).abs() / tol).max()
    assert far <= 1, f"states: {far:.2f} times the tolerance"
    # tokens: all see the first n keys; the last of T tokens see T - 1 more of the tail
    more = T - 1
    kp, vp = torch.cat([k, torch.zeros(more, heads * hd).to(dtype)]), torch.cat([v, torch.ones(more, heads * hd).to(dtype)])
    out = ops.chunk_attn(q.to(cuda), _paged(cuda, kp, vp, 64, T), 0, num_heads=heads, scale=1.0, left=n + T).double().cpu()[0]
    i = torch.arange(T)[:, None]
    want = weight * (v.double().sum(0) + i) / (1 + (n - 1 + i) * weight)
    far = ((out - want).abs() / ((3 * u + 2.0**-18 + n / 16 * 2.0**-24) * want)).max()
    assert far <= 1, f"tokens: {far:.2f} times the tolerance"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", [1, 50, 3000])
@pytest.mark.parametrize("T", [1, 20, 50])
def test_scores_of_minus_infinity(cuda, dtype, n, T):
    """Rows all of whose scores are -inf are NaN, as a softmax of them is; one finite score has the whole weight,
    wherever it is. Where no key is there, zeros stay zeros."""
    hd, heads = 64, 2
    q = torch.zeros(1, T, heads * hd).to(dtype)
    q[..., ::hd] = 1
    L = n + T - 1
    g = torch.Generator().manual_seed(n)
    v = torch.randn(L, heads * hd, generator=g).to(dtype)
    k = torch.zeros(L, heads * hd).to(dtype)
    k[:, ::hd] = -math.inf
    qd = q.to(cuda)
    lengths = torch.tensor([T - T // 3], dtype=torch.int32, device=cuda)

    def both(k, away=False):
        pages = _paged(cuda, k, v, 16, T)
        if away:
            pages.rows[0, 1:] = -1
        yield ops.chunk_attn(qd, pages, 0, num_heads=heads, lengths=lengths, left=L).cpu()[0]
        if not away:
            yield ops.cross_attn(qd, k[None].to(cuda), v[None].to(cuda), num_heads=heads).cpu()[0]

    m = T - T // 3
    print(f"[-inf] {dtype} n {n} T {T}", flush=True)
    tokens, texts = both(k)
    assert torch.isnan(tokens[:m]).all() and (tokens[m:] == 0).all() and torch.isnan(texts).all()
    (tokens,) = both(k, away=True)
    assert (tokens == 0).all()
    for at in {0, n // 2, n - 1}:
        one = k.clone()
        one[at] = 0
        tokens, texts = both(one)
        assert torch.equal(tokens[:m], v[at].expand(m, -1)) and (tokens[m:] == 0).all()
        assert torch.equal(texts, v[at].expand(T, -1))
    # a value that most tokens do not see is not finite: those rows are made again
    if T > 1:
        v[-1] = math.inf
        tokens, _ = both(k)
        assert torch.isnan(tokens[:m]).all() and (tokens[m:] == 0).all()


# fp16 ends at 2^16, and so do its products at 2^32
@pytest.mark.parametrize("dtype,bits", [(t, b) for b in (12, 20, 24, 25, 27, 29, 30, 32, 34, 36, 60, 100) for t in (F32, F16, BF16) if t is not F16 or b <= 30])
@pytest.mark.parametrize("n", [60, 3000])
def test_scores_far_past_fp32s_steps(cuda, dtype, bits, n):
    """Scores of up to 2^bits, of which fp32 knows steps of 2^(bits - 24) alone: the largest has the whole weight, two
    that are equal have half of it each, whatever their sign. All products are exact in fp32, the others 2^(bits - 7) lower.

    Halves are exact but for the output's rounding, u, the weights' and the sum's, 2 u, and fp32's: 2^-20."""
    hd, heads, u = 64, 2, HALF[dtype]
    g = torch.Generator().manual_seed(bits)
    v = torch.randn(n, heads * hd, generator=g).to(dtype)
    qd = 2.0 ** (bits // 2)
    top, low = 2.0 ** (bits - bits // 2), 2.0 ** (bits - bits // 2) - 2.0 ** (bits - bits // 2 - 7)
    for sign in (1, -1):
        for best in ([0], [n - 1], [n // 2, n - 2], [3, n // 3]):
            k = torch.zeros(n, heads * hd).to(dtype)
            k[:, ::hd] = low if sign == 1 else -top
            k[best, ::hd] = top if sign == 1 else -low
            want = v[best].double().mean(0)
            tol = (3 * u + 2.0**-20) * v[best].double().abs().mean(0) + 2.0**-30
            for T in (1, 40):
                q = torch.zeros(1, T, heads * hd).to(dtype)
                q[..., ::hd] = qd
                print(f"[far] {dtype} bits {bits} n {n} sign {sign} best {best} T {T}", flush=True)
                out = ops.cross_attn(q.to(cuda), k[None].to(cuda), v[None].to(cuda), num_heads=heads, scale=1.0).double().cpu()
                assert ((out - want).abs() <= tol).all(), f"states: {(out - want).abs().max()}"
                more = T - 1
                other = best[0] - 1 if best[0] else 1  # a key that is not one of the best: the step's own tokens have it, too
                pages = _paged(cuda, torch.cat([k, k[other].expand(more, -1)]), torch.cat([v, v[:1].expand(more, -1)]), 16, T)
                out = ops.chunk_attn(q.to(cuda), pages, 0, num_heads=heads, scale=1.0, left=n + T).double().cpu()
                assert ((out - want).abs() <= tol).all(), f"tokens: {(out - want).abs().max()}"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", [60, 700, 3000])
@pytest.mark.parametrize("T", [1, 40])
def test_scores_that_come_from_afar(cuda, dtype, n, T):
    """A third of the keys, first, last or every third, score -2^30 (fp16) or -2^36, the others 0: the output is the others' mean.

    Equal weights: the output's rounding, a weight's and the sum's, u each, fp32 sums over n keys in tiles of 16, 2^-18 as above."""
    hd, heads, u = 64, 2, HALF[dtype]
    g = torch.Generator().manual_seed(n)
    v = torch.randn(n, heads * hd, generator=g).to(dtype)
    q = torch.zeros(1, T, heads * hd).to(dtype)
    q[..., ::hd] = 2.0 ** (15 if dtype is F16 else 18)
    for away in (slice(0, n // 3), slice(n - n // 3, n), slice(0, n, 3)):
        k = torch.zeros(n, heads * hd).to(dtype)
        k[away, ::hd] = -q[0, 0, 0]
        near = torch.ones(n, dtype=torch.bool)
        near[away] = False
        want = v[near].double().mean(0)
        tol = (3 * u + 2.0**-18 + n / 16 * 2.0**-24) * v[near].double().abs().mean(0)
        print(f"[afar] {dtype} n {n} T {T} away {away}", flush=True)
        out = ops.cross_attn(q.to(cuda), k[None].to(cuda), v[None].to(cuda), num_heads=heads, scale=1.0).double().cpu()
        assert ((out - want).abs() <= tol).all(), f"states: {((out - want).abs() / tol).max()}"
        more = T - 1
        kp, vp = torch.cat([k, -q[0, :more].abs()]), torch.cat([v, v[:1].expand(more, -1)])
        out = ops.chunk_attn(q.to(cuda), _paged(cuda, kp, vp, 16, T), 0, num_heads=heads, scale=1.0, left=n + T).double().cpu()
        assert ((out - want).abs() <= tol).all(), f"tokens: {((out - want).abs() / tol).max()}"
