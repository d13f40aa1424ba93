"""Batch tables and adapters without a GPU: structures against the header, refusals
before a launch, the plain models against each other."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import paging
from parakeet_amd import _lib, ops
from parakeet_amd.modules import EncoderAdapters
from parakeet_amd.pool import DevicePagePool, PagePool
from tests._tables_model import RaggedPool, plan_model
from tests.test_abi import _struct_fields


@pytest.mark.parametrize(
    "cname,pyclass",
    [
        ("pk_page_step_args", _lib.PageStepArgs),
        ("pk_kv_append_slots_args", _lib.KvAppendSlotsArgs),
        ("pk_adapter_plan_args", _lib.AdapterPlanArgs),
        ("pk_adapter_linear_args", _lib.AdapterLinearArgs),
    ],
)
def test_struct_layout_matches_header(cname, pyclass):
    assert [f[0] for f in pyclass._fields_] == _struct_fields(cname)


def test_null_args():
    L = _lib.lib()
    for f in (L.pk_page_step, L.pk_kv_append_slots, L.pk_adapter_plan, L.pk_adapter_linear):
        assert f(None, None) == _lib.PK_ERR_INVALID
        assert "NULL" in _lib.last_error()


@pytest.mark.parametrize("left,chunk,P", [(70, 2, 16), (9, 3, 2), (0, 2, 4), (5, 1, 4)])
def test_ragged_model_is_the_host_pool_for_whole_chunks(left, chunk, P):
    rng = np.random.default_rng(left + P)
    host = PagePool(6, P, left, chunk)
    model = RaggedPool(6, P, left, chunk, range(host.num_pages))
    assert model.M == paging.max_pages(left, chunk, P) == host.max_pages
    for step in range(200):
        if rng.random() < 0.1:
            s = int(rng.integers(0, 6))
            host.reset_slot(s)
            model.reset([s])
        slots = rng.permutation(6)[: rng.integers(1, 7)].astype(np.int32)
        rows, place = model.advance(slots.tolist(), [chunk] * len(slots))
        np.testing.assert_array_equal(host.advance(slots), rows)
        pos = rows[:, :1] + np.arange(chunk)
        ring = rows[:, 1:]
        np.testing.assert_array_equal(place, np.take_along_axis(ring, pos // P % host.max_pages, 1) * P + pos % P)
    np.testing.assert_array_equal(host.free_list(), list(model.free))


def test_plan_model_covers_every_row_once():
    ids = np.array([3, -1, 0, 3, 3, 9, 0], dtype=np.int32)
    order, sorted_ids, tiles = plan_model(ids, 20, 5)
    assert sorted(order.tolist()) == list(range(140))
    covered = np.concatenate([np.arange(f, f + n) for a, f, n, _ in tiles if a >= 0])
    np.testing.assert_array_equal(covered, np.flatnonzero(sorted_ids >= 0))
    for a, f, n, _ in tiles:
        assert a < 0 or (set(sorted_ids[f : f + n]) == {a} and 0 < n <= 32)


def _page_args():
    a = _lib.PageStepArgs()
    a.device, a.batch, a.num_slots, a.num_pages, a.page_size, a.left, a.chunk = -1, 2, 4, 24, 16, 70, 2
    return a


@pytest.mark.parametrize(
    "field,value,what",
    [("page_size", 12, "power of two"), ("page_size", 0, "power of two"), ("left", -1, "left >= 0"), ("chunk", 0, "chunk"),
     ("num_slots", 0, "num_slots"), ("batch", -1, "batch >= 0"), ("num_pages", 23, "cannot hold"), ("num_pages", 1 << 28, "2\\^31 frames"),
     ("left", 2**31 - 1, "left >= 0"), (None, None, "NULL")],
)
def test_page_step_refusals(field, value, what):
    a = _page_args()
    if field:
        setattr(a, field, value)
    assert _lib.lib().pk_page_step(ctypes.byref(a), None) == _lib.PK_ERR_INVALID
    import re

    assert re.search(what, _lib.last_error())


def test_page_step_refuses_too_many_slots_and_short_rows():
    L = _lib.lib()
    a = _page_args()
    a.num_slots, a.num_pages = _lib.PAGE_STEP_MAX_SLOTS + 1, 6 * (_lib.PAGE_STEP_MAX_SLOTS + 1)
    assert L.pk_page_step(ctypes.byref(a), None) == _lib.PK_ERR_UNSUPPORTED
    a = _page_args()
    a.batch = _lib.PAGE_STEP_MAX_SLOTS + 1
    assert L.pk_page_step(ctypes.byref(a), None) == _lib.PK_ERR_UNSUPPORTED and "streams" in _lib.last_error()
    a = _page_args()
    buf = ctypes.create_string_buffer(64)  # never read: the calls are refused
    at = ctypes.addressof(buf)
    a.queue = a.head = a.appended = a.ring = a.slots = a.rows = a.slot_map = at
    a.rows_stride, a.slot_map_stride = 6, 2
    assert L.pk_page_step(ctypes.byref(a), None) == _lib.PK_ERR_INVALID and "rows_stride" in _lib.last_error()
    a.rows_stride, a.slot_map_stride = 7, 1
    assert L.pk_page_step(ctypes.byref(a), None) == _lib.PK_ERR_INVALID and "slot_map_stride" in _lib.last_error()


def test_append_slots_refusals():
    L = _lib.lib()
    a = _lib.KvAppendSlotsArgs()
    a.dtype, a.device, a.batch, a.chunk = _lib.DTYPE_F16, -1, 1, 4
    buf = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buf) + 15) & ~15
    p = a.pages
    p.k_pool = p.v_pool = at
    p.num_layers, p.num_pages, p.page_size, p.d_model, p.max_pages, p.rows_stride = 1, 8, 16, 512, 6, 7
    a.key = a.value = at
    assert L.pk_kv_append_slots(ctypes.byref(a), None) == _lib.PK_ERR_INVALID  # no slot map
    a.slot_map = at
    for field, value in (("key", at + 2), ("value", None), ("key_stride_t", 12), ("value_stride_b", -8), ("slot_map_stride_b", -1), ("batch", -1),
                         ("layer", 1), ("dtype", 9)):
        keep = getattr(a, field)
        setattr(a, field, value)
        assert L.pk_kv_append_slots(ctypes.byref(a), None) == _lib.PK_ERR_INVALID, field
        setattr(a, field, keep)
    p.num_pages = 1 << 28
    assert L.pk_kv_append_slots(ctypes.byref(a), None) == _lib.PK_ERR_INVALID


def test_plan_refusals():
    L = _lib.lib()
    a = _lib.AdapterPlanArgs()
    a.device, a.batch, a.frames, a.num_adapters, a.max_tiles = -1, 5, 2, 3, 3
    assert L.pk_adapter_plan(ctypes.byref(a), None) == _lib.PK_ERR_INVALID and "NULL" in _lib.last_error()
    for field, value, code in (("max_tiles", 2, _lib.PK_ERR_INVALID), ("frames", 0, _lib.PK_ERR_INVALID), ("num_adapters", 0, _lib.PK_ERR_INVALID),
                               ("batch", -1, _lib.PK_ERR_INVALID), ("batch", 1 << 30, _lib.PK_ERR_INVALID), ("batch", 1 << 23, _lib.PK_ERR_INVALID), ("max_tiles", 1 << 24, _lib.PK_ERR_INVALID),
                               ("num_adapters", _lib.ADAPTER_MAX + 1, _lib.PK_ERR_UNSUPPORTED)):
        keep = getattr(a, field)
        setattr(a, field, value)
        assert L.pk_adapter_plan(ctypes.byref(a), None) == code, field
        setattr(a, field, keep)
    assert L.pk_adapter_plan_tiles(5, 2, 3) == 3 and L.pk_adapter_plan_tiles(100, 14, 8) == 1400 // 32 + 8 and L.pk_adapter_plan_tiles(0, 2, 3) == 0


def test_adapter_linear_refusals():
    L = _lib.lib()
    a = _lib.AdapterLinearArgs()
    buf = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buf) + 15) & ~15
    a.dtype, a.device, a.rows, a.n, a.k, a.rank, a.num_adapters, a.max_tiles = _lib.DTYPE_F16, -1, 4, 128, 128, 16, 3, 3
    a.x_stride = a.weight_stride = a.out_stride = 128
    assert L.pk_adapter_linear(ctypes.byref(a), None) == _lib.PK_ERR_INVALID and "NULL" in _lib.last_error()
    for f in ("x", "weight", "a", "b", "scale", "order", "ids", "tiles", "workspace", "out"):
        setattr(a, f, at)
    bad, unsupported = _lib.PK_ERR_INVALID, _lib.PK_ERR_UNSUPPORTED
    for field, value, code in (("n", 100, unsupported), ("k", 96, unsupported), ("rank", 12, unsupported), ("rank", 136, unsupported), ("rank", 0, unsupported),
                               ("num_adapters", 0, unsupported), ("num_adapters", 513, unsupported), ("activation", 2, bad), ("rows", -1, bad),
                               ("max_tiles", -1, bad), ("x", at + 8, bad), ("order", None, bad), ("x_stride", 132, bad), ("weight_stride", 64, bad),
                               ("out_stride", 120, bad), ("out_stride", 1 << 30, bad), ("x_stride", 1 << 62, bad), ("dtype", 5, bad), ("weight", None, bad)):
        keep = getattr(a, field)
        setattr(a, field, value)
        assert L.pk_adapter_linear(ctypes.byref(a), None) == code, (field, value)
        setattr(a, field, keep)
    a.rows = 0
    assert L.pk_adapter_linear(ctypes.byref(a), None) == _lib.PK_OK
    assert L.pk_adapter_workspace_bytes(_lib.DTYPE_F16, 2000, 2048, 640, 16, 90) >= 2000 * 64 and L.pk_adapter_workspace_bytes(_lib.DTYPE_F16, 0, 64, 512, 16, 4) == 0


def test_cpu_tensors_are_refused():
    z = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    st = ops.PageState(z(12), z(2), torch.zeros(2, dtype=torch.int64), z(2, 6), page_size=16, left=70, chunk=2)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.page_step(st, z(2))
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.adapter_plan(z(2), 2, num_adapters=3)
    pool = torch.zeros(1, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.kv_append_slots(ops.PagedKV(pool, pool, z(1, 3), 2), 0, pool[0, 0, :4], pool[0, 0, :4], z(4))
    h = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.adapter_linear(h, h, None, ops.Adapters(h[None], h[None], torch.zeros(1)), ops.AdapterPlan(z(4), z(4), z(1, 4)))


def test_state_and_map_shapes_are_checked():
    z = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    A = torch.zeros(2, dtype=torch.int64)
    good = dict(page_size=16, left=70, chunk=2)
    for st in (
        ops.PageState(z(12).long(), z(2), A, z(2, 6), **good),
        ops.PageState(z(12), z(3), A, z(2, 6), **good),
        ops.PageState(z(12), z(2), A.int(), z(2, 6), **good),
        ops.PageState(z(12), z(2), A, z(2, 5), **good),
        ops.PageState(z(12), z(2), A, z(2, 6), page_size=0, left=70, chunk=2),
    ):
        with pytest.raises(ValueError):
            ops.page_step(st, z(2))
    pool = torch.zeros(1, 2, 16, 64, dtype=torch.float16)
    pages = ops.PagedKV(pool, pool, z(1, 3), 2)
    kv = torch.zeros(4, 64, dtype=torch.float16)
    for key, value, m, err in ((kv, kv, z(5), ValueError), (kv, kv, z(4).long(), ValueError), (kv.float(), kv, z(4), TypeError),
                               (kv[:, :32], kv, z(4), ValueError), (kv, kv, z(1, 2, 2), ValueError), (kv, kv, z(4, 2)[:, 0], ValueError)):
        with pytest.raises(err):
            ops.kv_append_slots(pages, 0, key, value, m)
    with pytest.raises(ValueError):
        ops.adapter_plan(z(2).long(), 2, num_adapters=3)


def test_device_pool_arguments():
    for kw, what in ((dict(page_size=12), "power of two"), (dict(chunk=0), "chunk"), (dict(num_pages=11), "cannot hold"),
                     (dict(page_order=[0] * 12), "permutation"), (dict(num_slots=_lib.PAGE_STEP_MAX_SLOTS + 1), "num_slots")):
        args = dict(num_slots=2, page_size=16, left=70, chunk=2, device="cpu") | kw
        with pytest.raises(ValueError, match=what):
            DevicePagePool(**args)
    p = DevicePagePool(2, 16, 70, 2, "cpu")
    for slots in ([0, 0], [2], [-1]):
        with pytest.raises(ValueError, match="distinct"):
            p.advance(slots)
    assert p.free_pages() == 12 and p.free_list().tolist() == list(range(12)) and p.slot_info(1)[0] == 0


def test_targets_may_be_an_iterator():
    class Layer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.self_attn = torch.nn.Module()
            self.self_attn.qkv = torch.nn.Linear(64, 192)

    encoder = torch.nn.Module()
    encoder.layers = torch.nn.ModuleList([Layer(), Layer()])
    bank = EncoderAdapters(encoder, num_adapters=3, rank=8, targets=iter(["self_attn.qkv"]))
    a, b = torch.randn(4, 64), torch.randn(192, 4)
    bank.load(2, {"layers.1.self_attn.qkv": (a, b)}, scale=0.5)
    kept = bank.banks[1]["self_attn.qkv"]
    assert torch.equal(kept.a[2, :4], a) and torch.equal(kept.b[2, :, :4], b) and not kept.a[2, 4:].any() and kept.scale.tolist() == [0, 0, 0.5]
    assert not bank.banks[0]["self_attn.qkv"].a.any()
    for i, weights, err in ((3, {}, IndexError), (0, {"layers.2.self_attn.qkv": (a, b)}, KeyError), (0, {"layers.0.self_attn.qkv": (b, a)}, ValueError)):
        with pytest.raises(err):
            bank.load(i, weights)
    bank.clear(2)
    assert not kept.a.any() and not kept.b.any() and not kept.scale.any()
