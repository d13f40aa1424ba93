"""Every form that the adapted projection's rule picks, against 64-bit products.

A form is the launches, the tile, the parts of K and what else has code of its own: the
bytes of a row of x and ranks up to 16 (one launch); ranks below 32 in the tiles whose h
goes through LDS; fp16 ranks past 64, whose h has a unit for each 64.  The tolerance is
that of the adapted projection's other tests (test_gpu_adapters), here from sums on the
device."""

import ctypes
import random

import pytest
import torch

from parakeet_amd import _lib, ops

from test_gpu_adapters import _make, _run

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
CUS = 256  # of the GPU that the rule was fitted on

# streams, frames, K, N, rank, adapters; rows end inside a tile
SHAPES = {
    "fp32": [
        (18, 1, 256, 64, 24, 3), (17, 1, 256, 64, 8, 7), (2, 14, 512, 64, 24, 6), (18, 1, 512, 64, 8, 3), (3, 7, 256, 2560, 32, 94),
        (17, 1, 256, 2560, 16, 5), (11, 3, 512, 1536, 24, 3), (17, 1, 512, 2560, 8, 3), (193, 1, 256, 640, 32, 8), (193, 1, 256, 640, 8, 83),
        (65, 1, 512, 1920, 24, 4), (7, 7, 512, 2560, 8, 28), (23, 7, 256, 1536, 24, 172), (23, 7, 256, 1536, 16, 124), (130, 1, 512, 1920, 24, 4),
        (129, 1, 512, 1920, 16, 9), (17, 1, 64, 64, 48, 36), (17, 1, 2048, 64, 64, 70), (17, 1, 64, 2560, 32, 20), (17, 1, 2048, 2560, 96, 51),
        (66, 1, 64, 2560, 96, 5), (193, 1, 2048, 1920, 128, 49), (6, 7, 64, 64, 8, 2), (134, 3, 2048, 1920, 40, 9), (115, 7, 192, 1920, 16, 23),
        (55, 7, 256, 2560, 64, 3), (44, 14, 2048, 2560, 16, 10), (278, 3, 2048, 1536, 128, 7), (129, 3, 64, 2560, 16, 100), (387, 1, 64, 2560, 96, 14),
        (179, 14, 320, 2560, 24, 15), (883, 3, 192, 2560, 128, 4), (2822, 1, 2048, 2560, 8, 39), (112, 14, 2048, 4096, 128, 3),
    ],
    "fp16": [
        (3, 7, 512, 64, 32, 22), (6, 3, 512, 64, 8, 9), (2, 14, 1024, 64, 24, 255), (6, 3, 1024, 64, 8, 5), (19, 1, 512, 2560, 32, 3),
        (17, 1, 512, 2560, 8, 5), (7, 14, 1024, 640, 24, 7), (6, 3, 1024, 2560, 8, 3), (27, 3, 512, 1536, 32, 11), (65, 1, 512, 1920, 16, 6),
        (27, 3, 1024, 1536, 32, 3), (97, 2, 1024, 640, 8, 5), (23, 7, 512, 1536, 32, 5), (23, 7, 512, 1536, 8, 165), (43, 3, 1024, 1920, 32, 4),
        (161, 1, 1024, 1536, 16, 6), (17, 1, 128, 64, 32, 5), (17, 1, 128, 64, 72, 112), (17, 1, 2048, 64, 32, 225), (17, 1, 2048, 64, 96, 10),
        (17, 1, 128, 2560, 40, 4), (17, 1, 128, 2560, 128, 25), (17, 1, 2048, 2560, 16, 68), (17, 1, 2048, 2560, 128, 106), (156, 1, 512, 2560, 8, 168),
        (73, 2, 1024, 2560, 72, 144), (612, 1, 2560, 320, 64, 5), (10, 7, 2048, 2560, 128, 4), (195, 1, 128, 1920, 8, 4), (92, 7, 2048, 1536, 8, 34),
        (65, 1, 64, 64, 8, 18), (65, 1, 64, 64, 48, 16), (22, 3, 64, 64, 96, 7), (321, 1, 2048, 1536, 8, 24), (321, 1, 2048, 1536, 32, 19),
        (321, 1, 2048, 1536, 96, 14), (22, 3, 64, 128, 8, 9), (5, 14, 64, 128, 32, 9), (12, 7, 64, 128, 72, 2), (802, 2, 256, 2560, 8, 19),
        (1608, 1, 256, 2560, 40, 7), (803, 2, 256, 2560, 128, 3), (1611, 1, 2048, 1920, 8, 78), (230, 7, 2048, 1920, 48, 9), (541, 3, 2048, 1920, 72, 7),
        (864, 3, 192, 4096, 24, 3), (1034, 2, 192, 4096, 64, 3), (2726, 1, 64, 4096, 128, 5), (1032, 2, 2048, 4096, 24, 32), (147, 14, 2048, 4096, 64, 6),
        (286, 1, 5120, 3584, 24, 2), (1231, 2, 320, 2560, 112, 4), (1834, 2, 128, 4096, 64, 3), (232, 7, 512, 2560, 56, 1), (44, 14, 128, 320, 8, 2),
        (229, 7, 2048, 2560, 16, 12), (440, 7, 64, 4096, 112, 2), (1538, 2, 192, 4096, 24, 1), (803, 2, 2048, 2560, 40, 13), (232, 7, 2048, 2560, 96, 2),
        (1628, 1, 512, 2560, 16, 1), (92, 7, 2048, 1536, 72, 3), (1032, 2, 128, 192, 80, 1),
    ],
    "bf16": [
        (6, 3, 512, 64, 24, 3), (17, 1, 512, 64, 8, 8), (2, 14, 1024, 64, 24, 240), (6, 3, 1024, 64, 8, 38), (19, 1, 512, 2560, 32, 3),
        (17, 1, 512, 2560, 16, 4), (194, 1, 1024, 320, 32, 7), (17, 1, 1024, 2560, 8, 3), (27, 3, 512, 1536, 32, 7), (193, 1, 512, 640, 16, 21),
        (196, 1, 1024, 640, 24, 3), (7, 7, 1024, 2560, 8, 79), (161, 1, 512, 1536, 24, 8), (23, 7, 512, 1536, 16, 8), (65, 2, 1024, 1920, 24, 8),
        (162, 1, 1024, 1536, 16, 4), (17, 1, 128, 64, 40, 6), (17, 1, 2048, 64, 8, 3), (17, 1, 128, 2560, 64, 117), (17, 1, 2048, 2560, 48, 104),
        (147, 1, 512, 2560, 8, 181), (7, 14, 2048, 1920, 128, 6), (14, 14, 128, 1920, 16, 9), (74, 7, 2048, 1920, 8, 10), (66, 1, 64, 64, 16, 4),
        (65, 1, 64, 64, 96, 56), (23, 14, 2048, 1536, 16, 6), (107, 3, 2048, 1536, 64, 11), (68, 1, 64, 128, 16, 4), (22, 3, 64, 128, 32, 3),
        (386, 7, 256, 1536, 8, 7), (808, 2, 256, 2560, 72, 4), (229, 7, 2048, 1920, 16, 8), (115, 14, 2048, 1920, 40, 64), (1028, 2, 256, 4096, 24, 32),
        (381, 7, 64, 4096, 128, 8), (2049, 1, 2048, 4096, 24, 4), (2050, 1, 2048, 4096, 48, 5),
    ],
}


def _form(dtype, rows, n, k, rank, tiles, cus=CUS):
    f = _lib.AdapterForm()
    _lib.check(_lib.lib().pk_adapter_linear_form(ops.dtype_code(DTYPES[dtype]), rows, n, k, rank, tiles, cus, ctypes.byref(f)), "form")
    elem = 4 if dtype == "fp32" else 2
    own = (k * elem, rank <= 16) if f.launches == 1 else (f.tile_rows >= 64 and rank < 32, dtype == "fp16" and rank > 64)
    return (f.launches, f.tile_rows, f.tile_columns, f.parts, *own)


def _tiles(B, T, G):
    return _lib.lib().pk_adapter_plan_tiles(B, T, G)


@pytest.mark.parametrize("dtype", DTYPES)
def test_shapes_cover_the_rule(dtype):
    """What 150,000 random sizes pick is in the list."""
    covered = {_form(dtype, B * T, N, K, r, _tiles(B, T, G)) for B, T, K, N, r, G in SHAPES[dtype]}
    rng = random.Random(11)
    for _ in range(150_000):
        T = rng.choice([1, 2, 7, 14])
        B = max(1, int(2 ** rng.uniform(0, 12)) // T)
        N, K = (64 * rng.choice([1, 2, 3, 4, 5, 8, 10, 16, 24, 30, 32, 40, 64]) for _ in range(2))
        r, G = 8 * rng.randint(1, 16), int(2 ** rng.uniform(0, 9))
        f = _form(dtype, B * T, N, K, r, _tiles(B, T, G))
        assert f in covered, (f, (B, T, K, N, r, G))


def test_form_refusals():
    f = _lib.AdapterForm()
    L = _lib.lib()
    for bad in ((0, 0, 64, 64, 8, 1), (0, 1, 96, 64, 8, 1), (0, 1, 64, 0, 8, 1), (0, 1, 64, 64, 0, 1), (0, 1, 64, 64, 8, -1)):
        assert L.pk_adapter_linear_form(*bad, CUS, ctypes.byref(f)) == _lib.PK_ERR_INVALID
    assert L.pk_adapter_linear_form(0, 1, 64, 64, 8, 1, CUS, None) == _lib.PK_ERR_INVALID


def _reference(x, w, bias, ad, ids, silu):
    """(y, tolerance) in 64 bits, as test_gpu_adapters has it."""
    T, dt = x.shape[1], x.dtype
    d = lambda t: t.double()  # noqa: E731
    K, r = x.shape[-1], ad.a.shape[1]
    x, w = d(x).view(-1, K), d(w)
    s, S = x @ w.T, x.abs() @ w.T.abs()
    if bias is not None:
        s, S = s + d(bias), S + d(bias).abs()
    part = {torch.float16: 2.0**-22, torch.bfloat16: 2.0**-16, torch.float32: 0.0}[dt]
    tol = torch.zeros_like(s)
    row_ids = ids.repeat_interleave(T)
    for g in ids.unique().tolist():
        if 0 <= g < ad.a.shape[0]:
            at = (row_ids == g).nonzero()[:, 0]
            A, Bm, sc = d(ad.a[g]), d(ad.b[g]), d(ad.scale[g])
            h, H = sc * (x[at] @ A.T), sc.abs() * (x[at].abs() @ A.T.abs())
            s[at] += h @ Bm.T
            S[at] += H @ Bm.T.abs()
            tol[at] += (part * h.abs() + (2.0**-36 * h.abs().amax(-1, keepdim=True) if dt == torch.float16 else 0.0)) @ Bm.T.abs()
    tol = tol + (2 * K + r + 8) * 2.0**-24 * S
    y = s
    if silu:
        y = s / (1 + torch.exp(-s))
        # the exponential's argument is off by 1.5 2^-24 of it, the other steps by 2^-20
        tol = 1.1 * tol + (2.0**-20 + 1.5 * 2.0**-24 * s.abs()) * y.abs()
    if dt != torch.float32:
        tol = tol + torch.finfo(dt).eps / 2 * (y.abs() + tol)
    return y, tol + (2.0**-25 if dt == torch.float16 else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,shape", [(d, s) for d in DTYPES for s in SHAPES[d]], ids=lambda v: v if isinstance(v, str) else "-".join(map(str, v)))
def test_every_form(cuda, dtype, shape):
    B, T, K, N, r, G = shape
    x, w, bias, ad, ids = _make(cuda, B, T, K, N, r, G, DTYPES[dtype], seed=B + N, bias=B % 2 == 0)
    assert _form(dtype, B * T, N, K, r, _tiles(B, T, G), 0) == _form(dtype, B * T, N, K, r, _tiles(B, T, G))
    clean = None
    for silu in (True, False):
        clean = _run(x, w, bias, ad, ids, silu)
        y, tol = _reference(x, w, bias, ad, ids, silu)
        err = (clean.double().view(y.shape) - y).abs()
        assert (err <= tol).all(), f"{float((err / tol).max()):.3f} of the tolerance"
    # an infinity of one adapter: its own rows of that column, and no bit of any other
    g = int(ids.max())
    if g < 0:
        return
    ad.b[g, N // 2, r - 1] = float("inf")
    got, own = _run(x, w, bias, ad, ids), ids == g
    assert not torch.isfinite(got[own][..., N // 2]).any()
    got[own, :, N // 2] = clean[own, :, N // 2]
    assert torch.equal(got, clean)
