"""Range and precision of h = scale x A^T between the adapters' two products, fp16.

fp16 ends at 65504 and 2^-24; h, and each part of a long K, is a 32-bit sum of any size.
Bound of h's rounding, with a row of h kept as high and low fp16 parts in units of a
power of two that puts its largest entry in [2^14, 2^15): 2^-22 |h|, or half a step of
fp16's subnormals, 2^-25, in those units; each of the high and the low part is rounded to
that step at most twice more where parts of K or groups of ranks are brought to one
unit, which holds down to 2^-38 of it: together below 2^-36 of the row's largest entry.
The sums are 32-bit: 2^-24 of the absolute sum for each of their terms (x has one
nonzero in a row where a test says so: a product with K has one term then).  The output
is rounded once, half of fp16's step: 2^-11 |y|, 2^-25 below its normal numbers."""

import pytest
import torch

from parakeet_amd import ops

from test_gpu_adapters import _check, _make, _run

pytestmark = pytest.mark.gpu

# rows in one launch; a few rows a tile; K in two parts; 64 ranks twice; large tiles
SHAPES = [
    (1, 1, 512, 512, 8, 1), (5, 2, 512, 512, 16, 3), (5, 2, 1024, 256, 32, 3), (20, 1, 640, 640, 24, 20), (9, 2, 2048, 512, 24, 4),
    (9, 2, 2048, 512, 128, 4), (60, 14, 4096, 1024, 32, 12), (60, 14, 4096, 1024, 16, 16), (128, 14, 1024, 1024, 128, 8),
    (256, 14, 1024, 4096, 64, 8), (256, 14, 512, 2048, 128, 8),
]


def _one_hot(x, value):
    """x with one nonzero in a row, in a column of its own."""
    K = x.shape[-1]
    rows = x.shape[0] * x.shape[1]
    y = torch.zeros_like(x).view(rows, K)
    at = torch.arange(rows, device=x.device)
    y[at, at * 37 % K] = value.to(x.dtype).expand(rows)
    return y.view(x.shape)


def _reference(x, w, bias, ad, ids, terms):
    """(y, tolerance) in 64 bits; `terms`: nonzero products a sum over K has."""
    c = lambda t: t.double().cpu()  # noqa: E731
    x, w, A, Bm, sc = c(x), c(w), c(ad.a), c(ad.b), c(ad.scale)
    r = A.shape[1]
    s, S = x @ w.T, x.abs() @ w.T.abs()
    if bias is not None:
        s, S = s + c(bias), S + c(bias).abs()
    part = torch.zeros_like(s)
    for b, g in enumerate(ids.tolist()):
        if 0 <= g < A.shape[0]:
            h, H = sc[g] * (x[b] @ A[g].T), sc[g].abs() * (x[b].abs() @ A[g].T.abs())
            s[b] += h @ Bm[g].T
            S[b] += H @ Bm[g].T.abs()
            part[b] += (2.0**-22 * h.abs() + 2.0**-36 * h.abs().amax(-1, keepdim=True)) @ Bm[g].T.abs()
    tol = part + (2 * terms + r + 8) * 2.0**-24 * S
    return s, tol + 2.0**-11 * (s.abs() + tol) + 2.0**-25


@pytest.mark.parametrize("B,T,K,N,r,G", SHAPES)
def test_small_h_against_large_b(cuda, B, T, K, N, r, G):
    """h near 2^-18: a subnormal fp16 number, of 6 bits and no low part."""
    x, w, bias, ad, ids = _make(cuda, B, T, K, N, r, G, torch.float16, seed=r)
    x = _one_hot(x, torch.tensor(2.0**-8, device=cuda))
    ad = ops.Adapters((ad.a * K**0.5 * 2.0**-10).half(), (ad.b * r**0.5 * 2.0**13).half(), ad.scale)
    w, bias = (w * 0.25).half(), None if bias is None else (bias * 0.25).half()
    _check(_run(x, w, bias, ad, ids), *_reference(x, w, bias, ad, ids, 1))


@pytest.mark.parametrize("B,T,K,N,r,G", SHAPES)
def test_large_h_against_small_b(cuda, B, T, K, N, r, G):
    """h near 100000 times a B of 1/1000: terms of order 100."""
    x, w, bias, ad, ids = _make(cuda, B, T, K, N, r, G, torch.float16, seed=r + 1)
    ad = ops.Adapters((ad.a * 100).half(), (ad.b * 1e-3).half(), torch.full_like(ad.scale, 1000.0))
    got = _run(x, w, bias, ad, ids)
    assert torch.isfinite(got).all()
    _check(got, *_reference(x, w, bias, ad, ids, K))


@pytest.mark.parametrize("B,T,K,N,r,G", SHAPES)
def test_halves_of_k_that_cancel(cuda, B, T, K, N, r, G):
    """The first half of K gives about 200000, the second the opposite."""
    x, w, bias, ad, ids = _make(cuda, B, T, K, N, r, G, torch.float16, seed=r + 2)
    x = x.abs()
    a = (ad.a + 400.0 / K).half()
    a[..., K // 2 :] -= 800.0 / K
    ad = ops.Adapters(a, ad.b, torch.full_like(ad.scale, 1250.0))
    ad.b.mul_(1e-3)
    got = _run(x, w, bias, ad, ids)
    assert torch.isfinite(got).all()
    _check(got, *_reference(x, w, bias, ad, ids, K))


@pytest.mark.parametrize("B,T,K,N,r,G", SHAPES)
@pytest.mark.parametrize("turn", [0, 1])
def test_ranks_of_many_magnitudes(cuda, B, T, K, N, r, G, turn):
    """Entries of a row of h from 2^-10 to 2^17, groups of ranks and parts of K that differ."""
    x, w, bias, ad, ids = _make(cuda, B, T, K, N, r, G, torch.float16, seed=r + 3)
    x = _one_hot(x, torch.tensor(0.75, device=cuda))
    e = torch.linspace(-10, 10, r, device=cuda).round()
    e = torch.exp2(e.flip(0) if turn else e)
    a = ad.a * K**0.5 * e[None, :, None]
    if turn:  # the columns of a part of K that a row's nonzero is not in give nothing
        a[..., K // 2 :] *= 2.0**-6
    ad = ops.Adapters(a.half(), (ad.b / e).half(), ad.scale * 100)
    _check(_run(x, w, bias, ad, ids), *_reference(x, w, bias, ad, ids, 1))


@pytest.mark.parametrize("B,T,K,N,r,G", SHAPES)
def test_an_infinity_among_large_entries(cuda, B, T, K, N, r, G):
    """An infinite entry of h gives its sign through B; entries past 65504 beside it, of
    the opposite sign, are finite."""
    x, w, bias, ad, ids = _make(cuda, B, T, K, N, r, G, torch.float16, seed=r + 4)
    x = x.abs()
    ids.zero_()
    ad.a.fill_(-100.0)
    ad.a[:, r - 1] = 1.0
    ad.a[:, r - 1, K - 1] = float("inf")
    ad.b.fill_(1.0)
    ad.b[:, 1::2, r - 1] = -1.0
    x[..., K - 1] = 1.0
    got = _run(x, w, bias, ad, ids)
    assert (got[..., 0::2] == float("inf")).all() and (got[..., 1::2] == -float("inf")).all()
