"""Head norms and rotation of new queries and keys on their way into the pages, against the
definition in 64 bits."""

import numpy as np
import pytest
import torch

from parakeet_amd import ops
from tests._attend_model import HALF, norm_rotate, pool_places

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _inv(n, base=10000.0):
    return base ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)


def _near(got, want, size, pos, inv, dtype, what):
    """One rounding to the type, and fp32's before it: 8 in a sum of squares over lanes, 3 in root
    and quotient, 2 products, 3 half steps of cosine and sine each (and 2^-24 turns, 4 half steps),
    2 products and a sum; half a step of the angle in 64 bits, here and in the reference."""
    far = 0.0 if inv is None else float(pos.double().abs().max() * inv.max()) * 2.0**-51
    tol = HALF[dtype] * want.abs() + (24 * 2.0**-24 + far) * size + (2.0**-25 if dtype is F16 else 1e-38)
    worst = ((got.double().cpu() - want).abs() / tol).max().item() if want.numel() else 0.0
    assert worst <= 1, f"{what}: {worst:.2f} times the tolerance"


def _run(cuda, dtype, hd, heads, kv_heads, B, T, P=16, rotary=None, interleaved=False, norm=True, given=False, far=5000, seed=0, eps=1e-6, skip=True):
    rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    D, per = kv_heads * hd, (T + 2 * P - 2) // P
    N = B * per + 1
    A = rng.integers(0, far, B)
    pages = rng.permutation(N)[: B * per].reshape(B, per)
    at = A[:, None] % P + np.arange(T)
    slot = np.take_along_axis(pages, at // P, 1) * P + at % P
    if skip:
        slot[rng.random((B, T)) < 0.2] = -1
        if B * T > 2:
            slot[0, 0] = N * P  # past the pages: left out
    x = torch.randn(B, T, (heads + 2 * kv_heads) * hd, generator=g) * 2
    x = x.to(dtype)
    q, k, v = x[..., : heads * hd], x[..., heads * hd : heads * hd + D], x[..., heads * hd + D :]
    qw, kw = ((1 + 0.3 * torch.randn(hd, generator=g)).to(dtype) for _ in range(2))
    inv = None if rotary == 0 else _inv(rotary or hd)
    pos = torch.from_numpy(A)[:, None] + torch.arange(T)
    if given:
        pos = torch.from_numpy(rng.integers(0, far, (B, T)))
    rows = torch.full((B + 1, 3), -1, dtype=torch.int32)
    rows[:B, 0] = torch.from_numpy(A)
    pools = [torch.randn(2, N, P, D, generator=g).to(dtype) for _ in range(2)]
    dev = [p.to(cuda) for p in pools]
    print(f"[norm] {dtype} hd {hd} heads {heads}/{kv_heads} B {B} T {T} P {P} rotary {rotary} {interleaved}", flush=True)
    xd = x.to(cuda)
    args = (xd[..., : heads * hd], xd[..., heads * hd : heads * hd + D], xd[..., heads * hd + D :])
    paged = ops.PagedKV(dev[0], dev[1], rows.to(cuda), 2)
    kw_args = dict(num_heads=heads, q_weight=qw.to(cuda) if norm else None, k_weight=kw.to(cuda) if norm else None,
                   inv_freq=None if inv is None else inv.to(cuda), positions=pos.int().to(cuda) if given else None, eps=eps, interleaved=interleaved)
    slots = torch.from_numpy(slot.astype(np.int32)).to(cuda)
    out = ops.qk_norm_append(*args, paged, 1, slots, **kw_args)
    torch.cuda.synchronize()
    split = lambda t: t.double().unflatten(-1, (-1, hd))  # noqa: E731
    wq, sq = norm_rotate(split(q), qw.double() if norm else None, pos, inv, eps, interleaved)
    wk, sk = norm_rotate(split(k), kw.double() if norm else None, pos, inv, eps, interleaved)
    _near(out, wq.flatten(-2), sq.flatten(-2), pos, inv, dtype, "queries")
    # keys and values at their places, everything else of the pools as it was
    place = pool_places(pools[0])
    for pool, got, new, size in ((pools[0], dev[0], wk.flatten(-2), sk.flatten(-2)), (pools[1], dev[1], None, None)):
        want = pool.clone()
        ok = (slot >= 0) & (slot < N * P)
        b, t = np.nonzero(ok)
        cells = place[1][torch.from_numpy(slot[b, t] // P), torch.from_numpy(slot[b, t] % P)]
        got = got.cpu()
        if new is None:
            want.view(-1)[cells] = v[b, t]
            assert torch.equal(got, want)
        else:
            _near(got.view(-1)[cells], new[b, t], size[b, t], pos, inv, dtype, "keys")
            got.view(-1)[cells] = 0
            want.view(-1)[cells] = 0
            assert torch.equal(got, want)
    return out, args, paged, slots, kw_args


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd,heads,kv_heads", [(64, 8, 8), (128, 8, 2), (64, 3, 1), (128, 5, 5), (64, 1, 1), (128, 32, 4)])
@pytest.mark.parametrize("B,T", [(1, 1), (3, 5), (7, 33)])
def test_heads_and_tokens(cuda, dtype, hd, heads, kv_heads, B, T):
    _run(cuda, dtype, hd, heads, kv_heads, B, T)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,rotary", [(64, 16), (64, 32), (128, 16), (128, 32), (128, 64), (128, 128), (64, 0)])
def test_rotations(cuda, dtype, interleaved, hd, rotary):
    _run(cuda, dtype, hd, 4, 2, 3, 9, rotary=rotary, interleaved=interleaved)
    _run(cuda, dtype, hd, 4, 2, 3, 9, rotary=rotary, interleaved=interleaved, norm=False, given=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("far", [1, 10**6, 2**31 - 100])
def test_far_positions(cuda, dtype, far):
    _run(cuda, dtype, 128, 2, 1, 5, 40, far=far)
    _run(cuda, dtype, 64, 2, 1, 5, 4, far=far, given=True, interleaved=True)


@pytest.mark.parametrize("P", [1, 4, 8, 64])
def test_page_sizes(cuda, P):
    _run(cuda, F16, 64, 3, 3, 4, 13, P=P)
    _run(cuda, F32, 128, 2, 1, 4, 13, P=P)


def test_many_tokens(cuda):
    _run(cuda, BF16, 128, 8, 2, 30, 101)
    _run(cuda, F16, 64, 8, 8, 2000, 1, far=10**5)


def test_zero_heads_and_values_that_are_not_finite(cuda):
    """A head of zeros stays zeros with eps, and is NaN without; an infinity stays in its head."""
    q = torch.zeros(1, 2, 128, dtype=F16, device=cuda)
    q[0, 1, 5] = float("inf")
    q[0, 1, 64:] = 1
    pool = torch.zeros(1, 1, 16, 64, dtype=F16, device=cuda)
    pages = ops.PagedKV(pool, pool.clone(), torch.zeros(1, 2, dtype=torch.int32, device=cuda), 1)
    slots = torch.tensor([[0, 1]], dtype=torch.int32, device=cuda)
    one = torch.ones(64, dtype=F16, device=cuda)
    call = lambda eps: ops.qk_norm_append(q, q[..., :64], q[..., 64:], pages, 0, slots, num_heads=2, q_weight=one, k_weight=one, eps=eps)  # noqa: E731
    out = call(1e-6)
    assert (out[0, 0] == 0).all() and torch.isnan(out[0, 1, 5]) and (out[0, 1, 64:] == 1).all()
    assert torch.isnan(call(0.0)[0, 0]).all()


def test_in_place_and_layouts(cuda):
    """The query itself as output, an output that is a view, another stream: the same bits."""
    out, args, pages, slots, kw = _run(cuda, BF16, 128, 4, 2, 5, 7)
    hold = torch.full((5, 8, 600), 7.0, dtype=BF16, device=cuda)
    got = ops.qk_norm_append(*args, pages, 1, slots, out=hold[:, :7, 8:520], **kw)
    assert torch.equal(got, out) and (hold[:, 7] == 7).all() and (hold[..., :8] == 7).all() and (hold[..., 520:] == 7).all()
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        there = ops.qk_norm_append(*args, pages, 1, slots, **kw)
    torch.cuda.current_stream(cuda).wait_stream(side)
    assert torch.equal(there, out)
    own = args[0]
    assert ops.qk_norm_append(own, *args[1:], pages, 1, slots, out=own, **kw) is own and torch.equal(own, out)
    assert ops.qk_norm_append(*(t[:, :0] for t in args), pages, 1, slots[:, :0], **kw).shape == (5, 0, 512)
