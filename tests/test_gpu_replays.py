"""Replays of a recorded encoder step between eager steps, resets and inspections: the
cache is in the state that an eager step leaves."""

import pytest
import torch

from parakeet_amd.modules.encoder import EncoderStepGraph

from test_gpu_request_tables import D, LY, T, _encoder

pytestmark = pytest.mark.gpu


def _states(cuda, B, device_pages, n=2):
    enc = _encoder(cuda, torch.float16)
    length = torch.full((B,), T, dtype=torch.int64, device=cuda)
    states = [enc.init_streaming_state(batch_size=B, device=cuda, dtype=torch.float16, device_pages=device_pages) for _ in range(n)]
    return enc, length, states


def _x(cuda, B, seed):
    return torch.randn(B, T, D, generator=torch.Generator().manual_seed(seed)).half().to(cuda)


def _reset(state):
    state.cache.reset()
    state.processed_frames.zero_()
    state.cache_lengths.zero_()


@pytest.mark.parametrize("device_pages", [False, True])
def test_window_after_a_reset_and_a_replay(cuda, device_pages):
    B = 3
    enc, length, (eager, replay) = _states(cuda, B, device_pages)
    graph = EncoderStepGraph(enc, replay, length)
    with torch.no_grad():
        for step in range(3):
            enc(_x(cuda, B, step), eager, length=length)
            graph(_x(cuda, B, step))
        _reset(eager)
        _reset(replay)
        with pytest.raises(RuntimeError, match="no step"):
            replay.cache.window(0)
        want, _ = enc(_x(cuda, B, 9), eager, length=length)
        assert torch.equal(graph(_x(cuda, B, 9)), want)
    for layer in range(LY):
        for a, b in zip(eager.cache.window(layer), replay.cache.window(layer)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("device_pages", [False, True])
def test_replay_after_half_a_step(cuda, device_pages):
    B = 2
    enc, length, (state,) = _states(cuda, B, device_pages, 1)
    graph = EncoderStepGraph(enc, state, length)
    with torch.no_grad():
        for step in range(2):
            graph(_x(cuda, B, step))
        kv = torch.zeros(B, T, D, dtype=torch.float16, device=cuda)
        state.cache.update_attn_cache(0, kv, kv)
        if device_pages:
            with pytest.raises(RuntimeError, match=r"after layers \[0\]"):
                graph(_x(cuda, B, 5))
            state.cache.update_attn_cache(1, kv, kv)
            graph(_x(cuda, B, 5))


@pytest.mark.parametrize("device_pages", [False, True])
def test_eager_steps_between_replays(cuda, device_pages):
    B = 3
    enc, length, (eager, mixed) = _states(cuda, B, device_pages)
    graph = EncoderStepGraph(enc, mixed, length)
    with torch.no_grad():
        for step in range(9):
            x = _x(cuda, B, step)
            want, _ = enc(x, eager, length=length)
            got = enc(x, mixed, length=length)[0] if step % 4 == 2 else graph(x)
            assert torch.equal(got, want), step
    assert eager.cache.pool.free_list().tolist() == mixed.cache.pool.free_list().tolist()
    for slot in range(B):
        assert eager.cache.pool.slot_info(slot)[0] == mixed.cache.pool.slot_info(slot)[0] == 9 * T
