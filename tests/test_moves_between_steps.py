"""ModelCache: forks and compactions are for the time between steps, whichever view opened the step."""

import pytest
import torch

from parakeet_amd import ops
from parakeet_amd.modules.cache import ModelCache

LAYERS = 3


class _Called(Exception):
    pass


@pytest.fixture
def cache(monkeypatch):
    """A cache whose tables' launches are stubs: a fork or compaction that is let through raises _Called."""
    cache = ModelCache(LAYERS, (70, 1), 64, 9, batch_size=4, device_pages=True)
    monkeypatch.setattr(cache.pool, "advance", lambda *a, **k: None)
    monkeypatch.setattr(cache.pool, "reset_all", lambda: None)
    monkeypatch.setattr(cache.pool, "reset_slot", lambda slot: None)

    def called(*args):
        raise _Called

    monkeypatch.setattr(ops, "page_fork", called)
    monkeypatch.setattr(ops, "page_compact", called)
    return cache


def _refused(cache):
    for call in (lambda: cache.fork([0], [1]), cache.compact):
        with pytest.raises(RuntimeError, match="step"):
            call()
    assert cache._base._moved == 0


def _allowed(cache):
    for call in (lambda: cache.fork([0], [1]), cache.compact):
        with pytest.raises(_Called):
            call()


def _layers(view, n=LAYERS):
    for layer in range(n):
        view._begin_layer(layer)


def test_an_open_step(cache):
    """A step that was opened and has no layer yet, some of them, all of them."""
    _allowed(cache)
    cache.open_step()
    _refused(cache)
    _layers(cache, 2)
    _refused(cache)
    cache._begin_layer(2)
    _allowed(cache)
    _layers(cache)
    _allowed(cache)


@pytest.mark.parametrize("make", [lambda c: c.view(2), lambda c: c.batch([3, 1])])
def test_an_open_step_of_a_view(cache, make):
    """The cache, the view and another view: while one of them is in a step, none moves pages."""
    view, other = make(cache), cache.batch([2, 0])
    view.open_step()
    for c in (cache, view, other):
        _refused(c)
    _layers(view)
    for c in (cache, view, other):
        _allowed(c)


def test_a_step_that_is_given_up(cache):
    """Its slots reset, or stepped again whole, pages move again."""
    view = cache.batch([3, 1])
    view.open_step()
    view.reset_slot(0)
    _refused(cache)
    view.reset_slot(1)
    _allowed(cache)
    view.open_step()
    cache.reset()
    _allowed(cache)
    view.open_step()
    again = cache.batch([1, 3])
    _layers(again)
    _allowed(cache)


def test_a_replayed_step(cache):
    """A replay opens and closes its step."""
    with cache.replaying():
        pass
    _allowed(cache)
    cache.open_step()
    with cache.replaying():
        pass
    _allowed(cache)


def test_stale_rows_are_not_given_out(cache):
    """`paged()` of a step from before the pages moved; of one that follows, and of a view without a step, as ever."""
    view, fresh = cache.batch([0, 2]), cache.batch([1])
    _layers(cache)
    _layers(view)
    cache.paged(), view.paged()
    cache._base._moved += 1  # as a fork or a compaction does
    for c in (cache, view):
        with pytest.raises(RuntimeError, match="moved"):
            c.paged()
    assert isinstance(fresh.paged(), ops.PagedKV)
    with cache.recording():
        cache.paged()
    cache.open_step()
    assert cache.paged().rows is cache._rows and cache.paged().left == 70
    with pytest.raises(RuntimeError, match="moved"):
        view.paged()
