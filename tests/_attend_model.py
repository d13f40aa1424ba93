"""Attention of a text decoder and head norms with rotation, restated in 64 bits, with how
far a kernel of a given type may be from them."""

import math

import torch

# half a step of a type relative to the value: what one rounding adds
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}


def attend(q, k, v, seen, scale, dtype):
    """q [T, hd], k and v [L, hd], seen [T, L] in float64 -> (out [T, hd], tolerance [T, hd]).

    The tolerance counts, with p the softmax and u half a step of the type:
      one rounding of the output                                       u |out|
      one rounding of each p before the product with v, and of the sum 2 u sum p |v|
      fp16: p below 2^-14 of the largest has steps of 2^-24            2^-25 pmax sum |v|
      the scores' fp32 sums: hd + 4 roundings of the partial sums, at most
      e = (hd + 4) 2^-24 scale sum |q k| in a score, 2 e in exp and its sum   2 (e^(2 e) - 1) sum p |v|
      fp32 sums over the keys, exp2 and the quotient: 2^-22 and 2^-24 for each doubling of the keys
      and each tile of 16 (running sums are rescaled once a tile)."""
    k, v = torch.where(seen.any(0)[:, None], k, 0.0), torch.where(seen.any(0)[:, None], v, 0.0)
    s = (q @ k.T) * scale
    s = torch.where(seen, s, -math.inf)
    some = seen.any(1)
    p = torch.where(some[:, None], torch.softmax(s, 1), 0.0)
    p = torch.where(seen, p, 0.0)
    out, mean = p @ v, p @ v.abs()
    u = HALF[dtype]
    e = (q.shape[1] + 4) * 2.0**-24 * scale * torch.where(seen, q.abs() @ k.abs().T, 0.0).amax(1, keepdim=True)
    e = e + 2.0**-23 * torch.where(seen, s, 0.0).abs().amax(1, keepdim=True)  # the product with scale and log2 e, twice rounded
    L = k.shape[0]
    tol = u * out.abs() + (2 * u + 2 * torch.expm1(2 * e) + 2.0**-22 + 2.0**-24 * (math.log2(L + 1) + L / 16)) * mean
    if dtype is torch.float16:
        tol = tol + 2.0**-25 * p.amax(1, keepdim=True) * torch.where(seen.any(0)[:, None], v.abs(), 0.0).sum(0) + 2.0**-25
    return out, tol + 1e-30


def norm_rotate(x, weight, pos, inv_freq, eps, interleaved):
    """x [..., H, hd] float64, pos [...] -> the normed and rotated heads, and the magnitude that a
    relative error of fp32 refers to."""
    hd = x.shape[-1]
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    y, size = x.clone(), x.abs()
    if inv_freq is not None:
        n = inv_freq.numel()
        i = torch.arange(n)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        f = (pos.double()[..., None] * inv_freq)[..., None, :]
        y[..., a] = x[..., a] * torch.cos(f) - x[..., b] * torch.sin(f)
        y[..., b] = x[..., b] * torch.cos(f) + x[..., a] * torch.sin(f)
        size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def pool_places(pool):
    """The element of a pool [Ly, N, P, D] at (layer, page, row, column), as an index tensor of its
    flat memory [Ly, N, P, D] (pages are column blocks of 64 bytes)."""
    Ly, N, P, D = pool.shape
    cb = math.gcd(D, 64 // pool.element_size())
    return torch.arange(pool.numel()).view(Ly, N, D // cb, P, cb).transpose(2, 3).reshape(Ly, N, P, D)


def fill_pages(rows, P, M, D, first, end, dtype, g, layer=1, layers=3, extra=2):
    """Pools [layers, N, P, D] of NaN, but for the positions first[b] .. end[b] - 1 of each row of the
    block table in `layer`; returns (k_pool, v_pool, k, v), k[b] and v[b] being [end[b] - first[b], D]."""
    pages = [int(x) for r in rows for x in r[1:] if x >= 0]
    N = max(pages, default=0) + 1 + extra
    pools, dense = [], []
    for _ in range(2):
        x = torch.full((layers, N, P, D), float("nan"), dtype=dtype)
        at = pool_places(x)
        out = []
        for b in range(len(rows)):
            pos = torch.arange(first[b], end[b])
            val = torch.randn(len(pos), D, generator=g).to(dtype)
            if len(pos):
                page = torch.as_tensor([int(rows[b][1 + int(p) // P % M]) for p in pos])
                x.view(-1)[at[layer, page, pos % P]] = val
            out.append(val)
        pools.append(x)
        dense.append(out)
    return (*pools, *dense)
