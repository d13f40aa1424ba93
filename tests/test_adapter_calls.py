"""Calls of the adapted projection that something follows or rewrites (derivatives,
traces, function transforms, autocast) are refused before anything else is looked at."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from parakeet_amd import ops
from parakeet_amd.modules.adapters import StepAdapters


class _Marked(torch.Tensor):
    pass


def _operands(device="cpu", dtype=torch.float32):
    x, w, bias = (torch.zeros(s, dtype=dtype, device=device) for s in ((2, 64), (64, 64), (64,)))
    ad = ops.Adapters(torch.zeros(1, 8, 64, dtype=dtype, device=device), torch.zeros(1, 64, 8, dtype=dtype, device=device), torch.zeros(1, device=device))
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)  # noqa: E731
    return x, w, bias, ad, ops.AdapterPlan(i32(2), i32(2), i32(1, 4))



@pytest.mark.parametrize("which", ["x", "weight", "bias", "a", "b", "scale"])
def test_forward_mode_and_subclasses(which):
    x, w, bias, ad, plan = _operands()
    ops_of = {"x": x, "weight": w, "bias": bias, "a": ad.a, "b": ad.b, "scale": ad.scale}

    def call(t):
        o = ops_of | {which: t}
        return ops.adapter_linear(o["x"], o["weight"], o["bias"], ops.Adapters(o["a"], o["b"], o["scale"]), plan)

    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(forward_ad.make_dual(ops_of[which], torch.ones_like(ops_of[which])))
        with pytest.raises(RuntimeError, match="HIP device"):  # no tangent: only the device is wrong
            call(ops_of[which])
    with pytest.raises(RuntimeError, match="plain tensors, got _Marked"):
        call(ops_of[which].as_subclass(_Marked))
    with pytest.raises(RuntimeError, match="HIP device"):
        call(torch.nn.Parameter(ops_of[which], requires_grad=False))


def test_traces():
    x, w, bias, ad, plan = _operands()
    call = lambda t: ops.adapter_linear(t, w, bias, ad, plan)  # noqa: E731
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, x)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(call)(x)


def test_traced_module():
    x, w, bias, ad, plan = _operands()
    step = StepAdapters(type("Banks", (), {"banks": [{"proj": ad}]})(), plan)
    lin = torch.nn.Linear(64, 64).requires_grad_(False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda t: step.linear(0, "proj", lin, t), x)


@pytest.mark.gpu
def test_transforms_on_the_device(cuda):
    x, w, bias, ad, plan = _operands(cuda)
    plan = ops.adapter_plan(torch.zeros(2, dtype=torch.int32, device=cuda), num_adapters=1)
    call = lambda t: ops.adapter_linear(t, w, bias, ad, plan)  # noqa: E731
    with torch.autocast("cuda", torch.bfloat16):
        with pytest.raises(RuntimeError, match="enabled=False"):
            call(x)
        with torch.autocast("cuda", enabled=False):
            assert call(x).dtype == torch.float32
        h = _operands(cuda, torch.bfloat16)
        assert ops.adapter_linear(*h[:4], plan).dtype == torch.bfloat16  # autocast's own dtype
    with pytest.raises(RuntimeError):
        torch.vmap(call)(x[None])
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (x,), (x,))
    with pytest.raises(RuntimeError, match="no backward"):
        torch.func.grad(lambda t: call(t).sum())(x)
