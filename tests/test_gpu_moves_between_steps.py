"""ModelCache on the GPU: a fork or a compaction in an open step is refused and changes nothing."""

import pytest
import torch

from parakeet_amd.modules.cache import ModelCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("viewed", [False, True])
def test_an_open_step(cuda, viewed):
    Ly, D, S, left = 2, 64, 4, 40
    cache = ModelCache(Ly, (left, 1), D, 9, batch_size=S, device=cuda, dtype=torch.float16, device_pages=True)
    view = cache.batch([3, 1, 0, 2]) if viewed else cache
    g = torch.Generator(device=cuda).manual_seed(0)
    frames = [[] for _ in range(Ly)]

    def step(layers):
        for layer in layers:
            x = torch.randn(S, 2, D, generator=g, device=cuda).half()
            frames[layer].append(x)
            k, v = view.update_attn_cache(layer, x, -x)
            want = torch.cat([torch.zeros(S, left, D, device=cuda).half(), *frames[layer]], 1)[:, -(left + 2) :]
            assert torch.equal(k, want) and torch.equal(v, -want)

    for _ in range(25):
        step(range(Ly))
    tables = lambda: [t.clone() for t in (cache.pool.state.queue, cache.pool.state.head, cache.pool.state.appended, cache.pool.state.ring)]  # noqa: E731
    view.open_step()
    for begun in (0, 1):
        before = tables()
        for call in (lambda: cache.fork([0], [1]), lambda: view.fork([0], [1]), cache.compact, view.compact):
            with pytest.raises(RuntimeError, match="step"):
                call()
        assert all(torch.equal(a, b) for a, b in zip(before, tables()))
        step([begun])
    view.fork([0], [1])
    for f in frames:
        for x in f:
            x[1] = x[0]
    view.compact()
    for _ in range(4):
        step(range(Ly))
