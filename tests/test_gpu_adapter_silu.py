"""SiLU of the adapted projection over the whole range of fp32 and bf16.

exp(-v) is 2^(-v log2 e): the product's and the constant's rounding are off by 2^-24 and
2^-25 of an exponent of |v| log2 e, so 1.5 2^-24 |v| of the value; the exponential, the
reciprocal and the other operations by a few units of 2^-23, below 2^-20 together (a
reciprocal down to 2^-128 is a subnormal number of 22 bits).  From -88.72 down exp(-v) is past
fp32's range and the output zero, as v / (1 + exp(-v)) is."""

import pytest
import torch

from parakeet_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K,rows", [(512, 16), (640, 600), (512, 4000)])
def test_silu_far_from_zero(cuda, dtype, K, rows):
    v = torch.linspace(-100.0, 100.0, rows * 64, device=cuda).to(dtype).view(rows, 64)
    x = torch.zeros(rows, K, dtype=dtype, device=cuda)
    x[:, :64] = v
    w = torch.eye(64, K, dtype=dtype, device=cuda)  # the output before SiLU is v itself
    ad = ops.Adapters(*(torch.zeros(1, *s, dtype=dtype, device=cuda) for s in ((8, K), (64, 8))), torch.zeros(1, device=cuda))
    plan = ops.adapter_plan(torch.full((rows,), -1, dtype=torch.int32, device=cuda), num_adapters=1)
    got = ops.adapter_linear(x, w, None, ad, plan, silu=True).double().cpu()
    v = v.double().cpu()
    y = v / (1 + torch.exp(-v))
    tol = y.abs() * (1.5 * 2.0**-24 * v.abs() + 2.0**-20)
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (y.abs() + tol)
    far = v < -88.72
    assert (((got - y).abs() <= tol) | far).all()
    assert (far & (got.abs() > y.abs() + tol)).sum() == 0
    normal = ~far & (v < -87.0)
    assert normal.any() and (got[normal] != 0).all()
