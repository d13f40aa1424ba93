"""Projections with low-rank adapters of many requests against 64-bit products.

Tolerance, from the operator's arithmetic, for an output y = act(s), s = sum of
products, S the sum of their absolute values with the two adapter products nested:
one rounding of y (eps/2 |y|, eps of the storage type); fp32 accumulation of at most
K + r + 3 terms and of h's K terms, (2 K + r + 8) 2^-24 S; h kept in two parts, its rest
below 2^-16 (bf16) or 2^-22 (fp16) of |h|, and in fp16 at most 2^-25 where the low part is
subnormal, times |b|.  SiLU has a slope of at most 1.1 and is evaluated to 2^-20 of its
value (one exponential and a division).  fp32 has no storage rounding and no parts."""

import numpy as np
import pytest
import torch

from parakeet_amd import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _make(cuda, B, T, K, N, r, G, dtype, seed=0, bias=True, scale=1.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    rnd = lambda *s, std=1.0: (torch.randn(s, generator=g, device=cuda) * std).to(dtype)  # noqa: E731
    x, w = rnd(B, T, K), rnd(N, K, std=K**-0.5)
    ad = ops.Adapters(rnd(G, r, K, std=K**-0.5), rnd(G, N, r, std=r**-0.5), (torch.rand(G, generator=g, device=cuda) + 0.5) * scale)
    ids = torch.randint(-1, G, (B,), generator=g, device=cuda).to(torch.int32)
    return x, w, rnd(N) if bias else None, ad, ids


def _reference(x, w, bias, ad, ids, silu):
    """(y, tolerance) in 64 bits, on the CPU."""
    T, dt = x.shape[1], x.dtype
    c = lambda t: t.double().cpu()  # noqa: E731
    x, w, A, Bm, sc = c(x), c(w), c(ad.a), c(ad.b), c(ad.scale)
    K, r = x.shape[-1], A.shape[1]
    s, S = x @ w.T, x.abs() @ w.T.abs()
    if bias is not None:
        s, S = s + c(bias), S + c(bias).abs()
    part = {torch.float16: 2.0**-22, torch.bfloat16: 2.0**-16, torch.float32: 0.0}[dt]
    floor = 2.0**-25 if dt == torch.float16 else 0.0
    tol = torch.zeros_like(s)
    for b, g in enumerate(ids.tolist()):
        if 0 <= g < A.shape[0]:
            h, H = sc[g] * (x[b] @ A[g].T), sc[g] * (x[b].abs() @ A[g].T.abs())
            s[b] += h @ Bm[g].T
            S[b] += H @ Bm[g].T.abs()
            tol[b] += (part * h.abs() + floor) @ Bm[g].T.abs()
    tol = tol + (2 * K + r + 8) * 2.0**-24 * S
    y = s
    if silu:
        y = s / (1 + torch.exp(-s))
        tol = 1.1 * tol + 2.0**-20 * y.abs()
    if dt != torch.float32:
        tol = tol + torch.finfo(dt).eps / 2 * (y.abs() + tol)
    return y, tol


def _check(got, want, tol):
    err = (got.double().cpu() - want).abs()
    worst = float((err / tol.clamp(min=1e-30)).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3f} of the tolerance"


def _run(x, w, bias, ad, ids, silu=False, **kw):
    plan = ops.adapter_plan(ids, x.shape[1], num_adapters=ad.a.shape[0])
    return ops.adapter_linear(x, w, bias, ad, plan, silu=silu, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,K,N,r,G", [
    (1, 1, 512, 512, 8, 1), (1, 2, 512, 2048, 16, 8), (5, 3, 64, 64, 8, 2), (17, 1, 640, 640, 24, 40), (61, 1, 1024, 1024, 16, 64),
    (40, 14, 512, 512, 32, 6), (128, 2, 512, 2048, 64, 20), (60, 14, 1024, 1024, 128, 4), (3, 14, 4096, 1024, 48, 3), (33, 1, 192, 320, 40, 512),
    (700, 1, 256, 128, 8, 300), (9, 14, 512, 64, 24, 3), (37, 3, 1024, 192, 32, 1), (150, 2, 512, 2048, 16, 16), (5, 1, 256, 64, 32, 2),
])
def test_against_64_bits(cuda, dtype, B, T, K, N, r, G):
    x, w, bias, ad, ids = _make(cuda, B, T, K, N, r, G, dtype, seed=B + K, bias=B % 2 == 1)
    for silu in (False, True):
        _check(_run(x, w, bias, ad, ids, silu), *_reference(x, w, bias, ad, ids, silu))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,T,K,N,r", [(100, 14, 512, 1024, 16), (300, 14, 512, 512, 16), (1000, 2, 1024, 2048, 32)])
def test_many_rows(cuda, dtype, B, T, K, N, r):
    x, w, bias, ad, ids = _make(cuda, B, T, K, N, r, 24, dtype, seed=B)
    _check(_run(x, w, bias, ad, ids, True), *_reference(x, w, bias, ad, ids, True))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,K,N,r,G", [(256, 14, 512, 2048, 96, 24), (256, 14, 512, 1024, 128, 100), (120, 7, 2048, 512, 40, 9), (500, 1, 1024, 2048, 72, 60)])
def test_wide_ranks_in_large_tiles(cuda, dtype, B, T, K, N, r, G):
    """Ranks whose h takes more than one turn through LDS, or ends inside one; and with an
    infinity in one adapter, which makes such tiles sum again, the other rows' bits."""
    x, w, bias, ad, ids = _make(cuda, B, T, K, N, r, G, dtype, seed=r)
    got = _run(x, w, bias, ad, ids)
    _check(got, *_reference(x, w, bias, ad, ids, False))
    g = int(ids[0])  # an adapter that the batch has
    ad.b[g, N // 2, r - 1] = float("inf")
    again, own = _run(x, w, bias, ad, ids), ids == g
    assert not torch.isfinite(again[own][..., N // 2]).any()
    assert torch.equal(again[~own], got[~own])
    again[own, :, N // 2] = got[own, :, N // 2]
    assert torch.equal(again, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["none", "one", "blocks", "bad"])
def test_mixtures(cuda, dtype, how):
    B, T, K, N, r, G = 70, 2, 128, 192, 16, 5
    x, w, bias, ad, ids = _make(cuda, B, T, K, N, r, G, dtype)
    i = torch.arange(B, device=cuda)
    ids = {"none": torch.full_like(ids, -1), "one": torch.full_like(ids, 3), "blocks": (i // 9 % G).to(torch.int32), "bad": (i - 30).to(torch.int32)}[how]
    got = _run(x, w, bias, ad, ids)
    _check(got, *_reference(x, w, bias, ad, ids, False))
    if how == "none":  # the shared projection alone
        zero = ops.Adapters(torch.zeros_like(ad.a), torch.zeros_like(ad.b), ad.scale)
        assert torch.equal(got, _run(x, w, bias, zero, ids))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,K,r", [(40, 1, 256, 16), (9, 14, 256, 16), (200, 2, 256, 16), (30, 1, 512, 16), (11, 14, 512, 8), (300, 14, 512, 32)])
def test_an_adapter_reaches_its_own_rows_alone(cuda, dtype, B, T, K, r):
    """Infinities and NaN in one adapter, or in one row, leave the other rows as they are."""
    x, w, bias, ad, _ = _make(cuda, B, T, K, 128, r, 4, dtype)
    ids = (torch.arange(B, device=cuda) * 7 % 5 - 1).to(torch.int32)
    clean = _run(x, w, bias, ad, ids)
    for what in ("a", "b", "scale"):
        for bad in (float("nan"), float("inf")):
            t = {k: getattr(ad, k).clone() for k in ("a", "b", "scale")}
            t[what][2] = bad
            got = _run(x, w, bias, ops.Adapters(**t), ids)
            own = ids == 2
            assert torch.equal(got[~own], clean[~own])
            assert not torch.isfinite(got[own]).any()
    y = x.clone()
    y[3, 0, 7] = float("nan")
    got = _run(y, w, bias, ad, ids)
    assert torch.isnan(got[3, 0]).all()
    got[3, 0] = clean[3, 0]
    assert torch.equal(got, clean)


def test_an_infinite_h_stays_infinite(cuda):
    """h past fp16's range is infinite, as one by one products leave it, and not NaN."""
    x, w, _, ad, ids = _make(cuda, 4, 2, 64, 64, 8, 1, torch.float16)
    ids.zero_()
    ad.scale.fill_(1e8)
    ad.b.fill_(1.0)
    ad.a[0] = 1.0
    x = x.abs()
    assert torch.isinf(_run(x, w, None, ad, ids)).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_out_and_strides(cuda, dtype):
    B, T, K, N, r, G = 12, 3, 128, 256, 8, 4
    x, w, bias, ad, ids = _make(cuda, B, T, K, N, r, G, dtype)
    want = _run(x, w, bias, ad, ids)
    wide = torch.zeros(N, K + 64, dtype=dtype, device=cuda)
    wide[:, :K] = w
    assert torch.equal(_run(x, wide[:, :K], bias, ad, ids), want)
    xw = torch.zeros(B, T, 2 * K, dtype=dtype, device=cuda)
    xw[..., K:] = x
    assert torch.equal(_run(xw[..., K:], w, bias, ad, ids), want)
    assert torch.equal(_run(x.transpose(0, 1).contiguous().transpose(0, 1), w, bias, ad, ids), want)
    odd = torch.zeros(x.numel() + 1, dtype=dtype, device=cuda)[1:].view(x.shape)
    odd.copy_(x)
    assert torch.equal(_run(odd, w, bias, ad, ids), want)
    guard = torch.full((B * T + 2, N), 7.0, dtype=dtype, device=cuda)
    out = guard[1:-1].view(B, T, N)
    assert _run(x, w, bias, ad, ids, out=out) is out and torch.equal(out, want)
    assert (guard[0] == 7).all() and (guard[-1] == 7).all()  # rows around the output are left as they were
    flat = ops.adapter_plan(ids.repeat_interleave(T), 1, num_adapters=G)
    assert torch.equal(ops.adapter_linear(x.view(B * T, K), w, bias, ad, flat).view(B, T, N), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_batch(cuda, dtype):
    x, w, bias, ad, ids = _make(cuda, 3, 2, 128, 64, 8, 2, dtype)
    assert _run(x[:0], w, bias, ad, ids[:0]).shape == (0, 2, 64)


def test_same_call_same_bits(cuda):
    x, w, bias, ad, ids = _make(cuda, 150, 2, 512, 1024, 16, 30, torch.bfloat16)
    first = _run(x, w, bias, ad, ids, True)
    for _ in range(3):
        assert torch.equal(_run(x, w, bias, ad, ids, True), first)


@pytest.mark.parametrize("dtype", DTYPES)
def test_recorded_twice_and_on_another_stream(cuda, dtype):
    """Two graphs and eager calls in turn: each has a workspace of its own."""
    sets = [_make(cuda, b, 2, 256, 512, 16, 6, dtype, seed=b) for b in (20, 75)]
    eager = [_run(*s, True) for s in sets]
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        aside = _run(*sets[1], True)
    torch.cuda.current_stream(cuda).wait_stream(side)
    assert torch.equal(aside, eager[1])
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_run(*s, True))
        graphs.append(g)
    for turn in range(4):
        ids = torch.roll(sets[0][4], turn)
        sets[0][4].copy_(ids)  # the next step's adapters
        for g in graphs:
            g.replay()
        want = _run(*sets[0], True)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], eager[1])


def test_refusals(cuda):
    x, w, bias, ad, ids = _make(cuda, 6, 2, 128, 64, 8, 2, torch.float16)
    plan = ops.adapter_plan(ids, 2, num_adapters=2)
    call = lambda x=x, w=w, bias=bias, ad=ad, plan=plan, **kw: ops.adapter_linear(x, w, bias, ad, plan, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="plan.order"):
        call(x=x[:5])
    with pytest.raises(ValueError, match="weight"):
        call(w=w[:, :64])
    with pytest.raises(ValueError, match="bias"):
        call(bias=bias[:32])
    with pytest.raises(ValueError, match="adapters must"):
        call(ad=ops.Adapters(ad.a.bfloat16(), ad.b, ad.scale))
    with pytest.raises(ValueError, match="adapters must"):
        call(ad=ops.Adapters(ad.a.transpose(1, 2), ad.b, ad.scale))
    with pytest.raises(ValueError, match="scale"):
        call(ad=ops.Adapters(ad.a, ad.b, ad.scale.half()))
    with pytest.raises(NotImplementedError, match="rank 4"):
        call(ad=ops.Adapters(ad.a[:, :4].contiguous(), ad.b[..., :4].contiguous(), ad.scale))
    with pytest.raises(NotImplementedError, match="multiples of 64"):
        y, v, c, b2, _ = _make(cuda, 6, 2, 96, 64, 8, 2, torch.float16)
        call(x=y, w=v, bias=c, ad=b2)
    with pytest.raises(ValueError, match="different devices"):
        call(ad=ops.Adapters(ad.a.cpu(), ad.b, ad.scale))
    with pytest.raises(ValueError, match="out must"):
        call(out=torch.empty(6, 2, 32, dtype=torch.float16, device=cuda))
    y, v, c, b2, _ = _make(cuda, 6, 2, 64, 64, 8, 2, torch.float16)
    for over in (y, v[:12].view(6, 2, 64)):
        with pytest.raises(ValueError, match="overlap"):
            call(x=y, w=v, bias=c, ad=b2, out=over)
    with pytest.raises(RuntimeError, match="no backward"):
        call(w=w.clone().requires_grad_())
    with pytest.raises(TypeError):
        call(x=x.double())
    with torch.no_grad():
        call(w=w.clone().requires_grad_())
    # a plan of another batch of the same size names rows of that batch: wrong rows, but none out of range
    junk = ops.AdapterPlan(torch.full_like(plan.order, 2**31 - 1), torch.full_like(plan.ids, 7), torch.full_like(plan.tiles, 2**30))
    call(plan=junk)
    torch.cuda.synchronize()
