"""The adapted encoder in 16-bit types against fp32 encoders with the adapters merged into
their weights, and recorded on host pages.

Bound: some 20 products, norms and softmaxes one after another, the 16-bit side rounding
each once and its residual beside it, 40 roundings of at most half a step of a value of
order 1: errors of a uniform distribution, half a step / sqrt(3) each, add as their squares,
and a branch has a gain of a few, at most 8: sqrt(40 / 3) 8 half steps, in the mean square.
fp32's own errors are 2^-13 of that.  An encoder with another adapter has to be past it."""

import copy
import math

import pytest
import torch

from parakeet_amd.modules.encoder import EncoderStepGraph

from test_gpu_request_tables import D, T, _adapters, _encoder, _same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_adapted_encoder_is_the_merged_encoders(cuda, dtype):
    enc = _encoder(cuda, dtype)
    ad, weights = _adapters(enc, 3, 16, 21)
    merged = []
    for w in weights + [{}]:
        m = copy.deepcopy(enc).float()
        for name, (a, b) in w.items():
            p = m.get_submodule(name).weight
            p.copy_((p.double().cpu() + 0.7 * b.to(dtype).double() @ a.to(dtype).double()).float())
        merged.append(m)
    ids = [2, -1, 0, 1, 2, 0]
    B = len(ids)
    state = enc.init_streaming_state(batch_size=B, device=cuda, dtype=dtype, device_pages=True)
    alone = [[m.init_streaming_state(batch_size=1, device=cuda, dtype=torch.float32) for m in merged] for _ in ids]
    dev_ids = torch.tensor(ids, dtype=torch.int32, device=cuda)
    g = torch.Generator().manual_seed(8)
    bound = math.sqrt(40 / 3) * 8 * torch.finfo(dtype).eps / 2
    one = torch.full((1,), T, dtype=torch.int64, device=cuda)
    rms = lambda e: float(e.double().square().mean().sqrt())  # noqa: E731
    with torch.no_grad():
        for step in range(9):
            x = torch.randn(B, T, D, generator=g).to(dtype).to(cuda)
            got, state = enc(x, state, length=one.expand(B).contiguous(), adapters=ad.step(dev_ids, T))
            for b, i in enumerate(ids):
                for j, m in enumerate(merged):
                    want, alone[b][j] = m(x[b : b + 1].float(), alone[b][j], length=one)
                    err = rms(got[b].float() - want[0])
                    if j == i % len(merged):  # -1: the last one, without an adapter
                        assert err < bound, (step, b, err, bound)
                    else:
                        assert err > bound, (step, b, j, err, bound)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_recorded_on_host_pages(cuda, dtype):
    """Host pages are advanced before each replay; adapters and their numbers change between."""
    enc = _encoder(cuda, dtype)
    ad, weights = _adapters(enc, 3, 8, 22)
    B = 5
    length = torch.full((B,), T, dtype=torch.int64, device=cuda)
    eager, replay = (enc.init_streaming_state(batch_size=B, device=cuda, dtype=dtype) for _ in range(2))
    ids = torch.zeros(B, dtype=torch.int32, device=cuda)
    graph = EncoderStepGraph(enc, replay, length, adapters=ad, adapter_ids=ids)
    g = torch.Generator().manual_seed(19)
    with torch.no_grad():
        for step in range(8):
            x = torch.randn(B, T, D, generator=g).to(dtype).to(cuda)
            ids.copy_(torch.randint(-1, 4, (B,), generator=g).to(torch.int32))
            if step == 5:
                ad.load(1, weights[2], 0.3)
            want, _ = enc(x, eager, length=length, adapters=ad.step(ids, T))
            assert torch.equal(graph(x), want), step
            _same(eager, replay)
