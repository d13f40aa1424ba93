"""A text decoder's operators without a GPU: structures against the header, refusals before a
launch, the plain models against each other."""

import ctypes
import math

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from parakeet_amd import _lib, ops
from parakeet_amd.modules import ModelCache
from parakeet_amd.pool import DevicePagePool
from tests._attend_model import attend, fill_pages, norm_rotate, pool_places
from tests._page_moves_model import compact, fork
from tests._tables_model import RaggedPool
from tests.test_abi import _struct_fields

STRUCTS = [("pk_page_fork_args", _lib.PageForkArgs), ("pk_page_compact_args", _lib.PageCompactArgs), ("pk_kv_move_pages_args", _lib.KvMovePagesArgs),
           ("pk_qk_norm_append_args", _lib.QkNormAppendArgs), ("pk_chunk_attn_args", _lib.ChunkAttnArgs), ("pk_cross_attn_args", _lib.CrossAttnArgs)]


@pytest.mark.parametrize("cname,pyclass", STRUCTS)
def test_struct_layout_matches_header(cname, pyclass):
    assert [f[0] for f in pyclass._fields_] == _struct_fields(cname)


def test_null_args():
    L = _lib.lib()
    for f in (L.pk_page_fork, L.pk_page_compact, L.pk_kv_move_pages, L.pk_qk_norm_append, L.pk_chunk_attn, L.pk_cross_attn):
        assert f(None, None) == _lib.PK_ERR_INVALID
        assert "NULL" in _lib.last_error()


# ---------------------------------------------------------------------------
# refusals of the C entry points: every check comes before the device is looked at


def _memory():
    """Some 16-byte aligned host memory: only its address is used."""
    buf = ctypes.create_string_buffer(4096)
    return buf, (ctypes.addressof(buf) + 15) & ~15


def _layout(at):
    L = _lib.PagedLayout()
    L.k_pool = L.v_pool = L.rows = at
    L.num_layers, L.num_pages, L.page_size, L.d_model, L.rows_stride, L.max_pages = 2, 40, 16, 256, 7, 6
    return L


def _fork_args(at):
    a = _lib.PageForkArgs()
    a.device, a.batch, a.num_slots, a.num_pages, a.page_size, a.left, a.chunk = -1, 2, 4, 24, 16, 70, 2
    for f in ("queue", "head", "appended", "ring", "src", "dst", "pairs", "count"):
        setattr(a, f, at)
    return a


def _compact_args(at):
    a = _lib.PageCompactArgs()
    a.device, a.num_slots, a.num_pages, a.max_pages, a.capacity = -1, 4, 24, 6, 12
    for f in ("queue", "head", "ring", "pairs", "count"):
        setattr(a, f, at)
    return a


def _move_args(at):
    a = _lib.KvMovePagesArgs()
    a.device, a.dtype, a.pages, a.capacity, a.pairs, a.count = -1, 1, _layout(at), 4, at, at
    return a


def _norm_args(at):
    a = _lib.QkNormAppendArgs()
    a.device, a.dtype, a.pages, a.batch, a.chunk, a.num_heads, a.head_dim, a.rotary, a.eps = -1, 1, _layout(at), 2, 3, 8, 64, 64, 1e-6
    for f in ("query", "key", "value", "out", "q_weight", "k_weight", "inv_freq", "slot_map"):
        setattr(a, f, at)
    return a


def _chunk_args(at):
    a = _lib.ChunkAttnArgs()
    a.device, a.dtype, a.pages, a.batch, a.chunk, a.num_heads, a.head_dim, a.left, a.scale = -1, 1, _layout(at), 2, 3, 8, 64, 70, 0.125
    a.query = a.out = a.workspace = at
    return a


def _cross_args(at):
    a = _lib.CrossAttnArgs()
    a.device, a.dtype, a.batch, a.chunk, a.states, a.num_heads, a.kv_heads, a.head_dim, a.scale = -1, 1, 2, 3, 70, 8, 4, 64, 0.125
    a.query = a.out = a.key = a.value = a.workspace = at
    return a


CALLS = {"fork": ("pk_page_fork", _fork_args), "compact": ("pk_page_compact", _compact_args), "move": ("pk_kv_move_pages", _move_args),
         "norm": ("pk_qk_norm_append", _norm_args), "chunk": ("pk_chunk_attn", _chunk_args), "cross": ("pk_cross_attn", _cross_args)}
BAD = [
    ("fork", "page_size", 12, "power of two"), ("fork", "left", -1, "left"), ("fork", "chunk", 0, "chunk"), ("fork", "num_pages", 23, "cannot hold"),
    ("fork", "num_pages", 1 << 30, "2\\^30"), ("fork", "batch", -1, "batch"), ("fork", "batch", 5, "5 pairs for 4 slots"), ("fork", "queue", None, "NULL"),
    ("fork", "head", None, "NULL"), ("fork", "appended", None, "NULL"), ("fork", "ring", None, "NULL"), ("fork", "src", None, "NULL"),
    ("fork", "dst", None, "NULL"), ("fork", "pairs", None, "NULL"), ("fork", "count", None, "NULL"), ("fork", "left", 2**31 - 1, "left"),
    ("compact", "num_slots", 0, "num_slots"), ("compact", "max_pages", 0, "max_pages"), ("compact", "num_pages", 23, "cannot hold"),
    ("compact", "num_pages", 1 << 30, "2\\^30"), ("compact", "capacity", 11, "needs 12"), ("compact", "queue", None, "NULL"),
    ("compact", "head", None, "NULL"), ("compact", "ring", None, "NULL"), ("compact", "pairs", None, "NULL"), ("compact", "count", None, "NULL"),
    ("move", "dtype", 7, "dtype"), ("move", "capacity", -1, "capacity"), ("move", "pairs", None, "NULL"), ("move", "count", None, "NULL"),
    ("move", "pages.k_pool", None, "NULL"), ("move", "pages.num_layers", 0, "layers"), ("move", "pages.page_size", 0, "page_size"),
    ("move", "pages.d_model", 0, "d_model"), ("move", "pages.num_layers", 2**31 - 1, "2\\^31 units"), ("move", "pages.k_pool", 8, "aligned"),
    ("norm", "dtype", 3, "dtype"), ("norm", "head_dim", 96, "head_dim 96"), ("norm", "pages.page_size", 3, "power of two"), ("norm", "layer", 2, "layer 2"),
    ("norm", "layer", -1, "layer -1"), ("norm", "batch", -1, "batch"), ("norm", "chunk", -2, "chunk"), ("norm", "num_heads", 0, "num_heads"),
    ("norm", "rotary", 24, "rotary 24"), ("norm", "rotary", 128, "rotary 128"), ("norm", "rotary", 8, "rotary 8"), ("norm", "eps", -1.0, "eps"),
    ("norm", "eps", math.nan, "eps"), ("norm", "eps", math.inf, "eps"), ("norm", "query", None, "query is NULL"), ("norm", "key", None, "key is NULL"),
    ("norm", "value", None, "value is NULL"), ("norm", "out", None, "out is NULL"), ("norm", "slot_map", None, "NULL"), ("norm", "inv_freq", None, "NULL"),
    ("norm", "query_stride_t", 4, "aligned"), ("norm", "key_stride_b", -8, "aligned"), ("norm", "pages.d_model", 96, "whole heads"),
    ("norm", "pages.rows", None, "NULL"), ("norm", "slot_map_stride_b", -1, "negative"), ("norm", "pages.num_pages", 1 << 28, "2\\^31"),
    ("norm", "pages.v_pool", None, "pools"), ("norm", "chunk", 2**31 - 1, "2\\^24|2\\^31"),
    ("chunk", "dtype", -1, "dtype"), ("chunk", "head_dim", 32, "head_dim 32"), ("chunk", "num_heads", 6, "whole groups"), ("chunk", "batch", -1, "batch"),
    ("chunk", "scale", 0.0, "scale"), ("chunk", "scale", math.nan, "scale"), ("chunk", "scale", math.inf, "scale"), ("chunk", "left", -1, "window"),
    ("chunk", "left", 79, "do not hold"), ("chunk", "pages.rows_stride", 6, "rows_stride 6"), ("chunk", "pages.rows", None, "rows is NULL"),
    ("chunk", "query", None, "query is NULL"), ("chunk", "out", None, "out is NULL"), ("chunk", "query", 8, "aligned"), ("chunk", "layer", 2, "layer 2"),
    ("chunk", "pages.k_pool", None, "pools"), ("chunk", "pages.page_size", 48, "power of two"), ("chunk", "pages.max_pages", 0, "rows_stride|window"),
    ("cross", "dtype", 9, "dtype"), ("cross", "head_dim", 80, "head_dim 80"), ("cross", "kv_heads", 3, "whole groups"), ("cross", "kv_heads", 0, "whole groups"),
    ("cross", "states", -1, "states"), ("cross", "key", None, "key is NULL"), ("cross", "value", None, "value is NULL"), ("cross", "scale", -1.0, "scale"),
    ("cross", "key_stride_t", 12, "aligned"), ("cross", "value", 8, "aligned"), ("cross", "batch", -3, "batch"), ("cross", "out_stride_b", -8, "aligned"),
    ("cross", "chunk", 2**31 - 1, "rows"),
]


@pytest.mark.parametrize("which,field,value,what", BAD)
def test_refusals(which, field, value, what):
    import re

    keep, at = _memory()
    name, make = CALLS[which]
    a = make(at)
    owner, _, leaf = field.rpartition(".")
    owner = getattr(a, owner) if owner else a
    setattr(owner, leaf, at + value if value == 8 and leaf in ("query", "value", "k_pool") else value)
    assert getattr(_lib.lib(), name)(ctypes.byref(a), None) in (_lib.PK_ERR_INVALID, _lib.PK_ERR_UNSUPPORTED)
    assert re.search(what, _lib.last_error()), _lib.last_error()
    del keep


@pytest.mark.parametrize("which", ["move", "norm", "chunk", "cross"])
def test_nothing_to_do(which):
    """An empty call is done without a look at its tensors."""
    name, make = CALLS[which]
    a = make(0)
    a.pages = _layout(_memory()[1]) if hasattr(a, "pages") else None
    setattr(a, "capacity" if which == "move" else "batch", 0)
    assert getattr(_lib.lib(), name)(ctypes.byref(a), None) == _lib.PK_OK
    if which in ("norm", "chunk", "cross"):
        a.batch, a.chunk = 2, 0
        assert getattr(_lib.lib(), name)(ctypes.byref(a), None) == _lib.PK_OK


# ---------------------------------------------------------------------------
# refusals of the tensor calls


def _pages(dtype=torch.float16, D=128, device="cpu"):
    pool = torch.zeros(1, 8, 16, D, dtype=dtype, device=device)
    return ops.PagedKV(pool, pool.clone(), torch.zeros(2, 7, dtype=torch.int32, device=device), 6)


def _tensors(dtype=torch.float16):
    z = lambda *s: torch.zeros(s, dtype=dtype)  # noqa: E731
    return z(2, 3, 256), z(2, 3, 128), z(2, 3, 128), torch.zeros(2, 3, dtype=torch.int32)


def _calls(dtype=torch.float16):
    q, k, v, slots = _tensors(dtype)
    pages = _pages(dtype)
    return {
        "qk_norm_append": lambda query=q, **kw: ops.qk_norm_append(query, kw.pop("key", k), kw.pop("value", v), kw.pop("pages", pages), 0,
                                                                   kw.pop("slot_map", slots), num_heads=kw.pop("num_heads", 4), **kw),
        "chunk_attn": lambda query=q, **kw: ops.chunk_attn(query, kw.pop("pages", pages), 0, num_heads=kw.pop("num_heads", 4), **kw),
        "cross_attn": lambda query=q, **kw: ops.cross_attn(query, kw.pop("key", k), kw.pop("value", v), num_heads=kw.pop("num_heads", 4), **kw),
    }


class _Marked(torch.Tensor):
    pass


ALL = ["qk_norm_append", "chunk_attn", "cross_attn"]


@pytest.mark.parametrize("name", ALL)
def test_cpu_tensors(name):
    with pytest.raises(RuntimeError, match="HIP device"):
        _calls()[name]()


@pytest.mark.parametrize("name", ALL)
def test_gradients_and_transforms(name):
    call = _calls(torch.float32)[name]
    q = torch.zeros(2, 3, 256, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward pass"):
        call(q)
    with torch.no_grad(), pytest.raises(RuntimeError, match="HIP device"):
        call(q)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        call(forward_ad.make_dual(q.detach(), torch.ones_like(q)))
    with pytest.raises(RuntimeError, match="plain tensors"):
        call(q.detach().as_subclass(_Marked))


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("kw,error,what", [
    ({"query": torch.zeros(2, 256, dtype=torch.float16)}, ValueError, "query must be"),
    ({"num_heads": 3}, ValueError, "query must be"),
    ({"num_heads": 8}, NotImplementedError, "heads of 64 and 128"),
    ({"num_heads": 0}, ValueError, "query must be"),
    ({"query": torch.zeros(2, 3, 512, dtype=torch.float16)[..., ::2]}, ValueError, "contiguous and 16-byte"),
    ({"query": torch.zeros(2, 3, 260, dtype=torch.float16)[..., 4:]}, ValueError, "contiguous and 16-byte"),
])
def test_queries(name, kw, error, what):
    with pytest.raises(error, match=what):
        _calls()[name](**kw)


@pytest.mark.parametrize("name,kw,error,what", [
    ("qk_norm_append", {"pages": _pages(torch.bfloat16)}, TypeError, "pages dtype"),
    ("qk_norm_append", {"pages": _pages(D=96)}, ValueError, "whole heads"),
    ("qk_norm_append", {"key": torch.zeros(2, 3, 64, dtype=torch.float16)}, ValueError, "key"),
    ("qk_norm_append", {"value": torch.zeros(2, 3, 128)}, TypeError, "value"),
    ("chunk_attn", {"pages": _pages(torch.bfloat16)}, TypeError, "pages dtype"),
    ("chunk_attn", {"pages": _pages(D=96)}, ValueError, "whole heads"),
    ("cross_attn", {"key": torch.zeros(2, 3, 96, dtype=torch.float16)}, ValueError, "whole heads"),
    ("cross_attn", {"key": torch.zeros(1, 3, 128, dtype=torch.float16)}, ValueError, "key"),
    ("cross_attn", {"value": torch.zeros(2, 4, 128, dtype=torch.float16)}, ValueError, "value"),
    ("cross_attn", {"key": torch.zeros(2, 3, 128)}, TypeError, "key"),
])
def test_operands(name, kw, error, what):
    with pytest.raises(error, match=what):
        _calls()[name](**kw)


def test_page_moves_on_the_cpu():
    st = ops.PageState(torch.arange(12).int(), torch.tensor([0, 12]).int(), torch.zeros(2).long(), torch.full((2, 6), -1).int(), 16, 70, 2)
    one = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.page_fork(st, one, one), lambda: ops.page_compact(st),
                 lambda: ops.kv_move_pages(torch.zeros(1, 2, 2, 8), torch.zeros(1, 2, 2, 8), ops.PageMoves(torch.zeros(1, 2).int(), one))):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
    for pairs, count in ((torch.zeros(1, 3).int(), one), (torch.zeros(2).int(), one), (torch.zeros(1, 2), one), (torch.zeros(1, 2).int(), torch.zeros(2).int())):
        with pytest.raises(ValueError, match="moves"):
            ops.kv_move_pages(torch.zeros(1, 2, 2, 8), torch.zeros(1, 2, 2, 8), ops.PageMoves(pairs, count))


@pytest.mark.parametrize("src,dst,what", [([0], [0], "both"), ([0, 1], [2], "as many"), ([9], [1], "slots must be in"), ([0, 0], [1, 1], "distinct"), ([0], [-1], "distinct")])
def test_pool_forks_refused(src, dst, what):
    with pytest.raises(ValueError, match=what):
        DevicePagePool(4, 16, 70, 2, "cpu").fork(src, dst)


def test_cache_forks_refused():
    host = ModelCache(1, (70, 1), 64, 9, batch_size=4)
    for call in (lambda: host.fork([0], [1]), host.compact):
        with pytest.raises(RuntimeError, match="device_pages"):
            call()
    cache = ModelCache(1, (70, 1), 64, 9, batch_size=4, device_pages=True)
    with pytest.raises(ValueError, match="rows must be in"):
        cache.view(2).fork([0], [2])
    with cache.recording(), pytest.raises(RuntimeError, match="not recorded"):
        cache.compact()


# ---------------------------------------------------------------------------
# the models


def test_moves_keep_what_streams_hold():
    """Forks and compactions of the model: pages are disjoint, and carry their frames along."""
    rng = np.random.default_rng(0)
    S, P, left, chunk = 9, 4, 11, 3
    model = RaggedPool(S, P, left, chunk, rng.permutation(S * 5 + 4))
    total, data, frames = len(model.free), {}, [[] for _ in range(S)]
    for turn in range(200):
        batch, lengths = rng.permutation(S)[:5], rng.integers(0, chunk + 1, 5)
        _, place = model.advance(batch.tolist(), lengths.tolist())
        for s, n, at in zip(batch, lengths, place):
            for t in range(n):
                data[int(at[t])] = (turn, int(s), t)
                frames[s].append((turn, int(s), t))
        moves = []
        if turn % 5 == 0:
            both = rng.permutation(S)
            moves = fork(model, both[4:7].tolist(), both[:3].tolist())
            for s, d in zip(both[4:7], both[:3]):
                frames[d] = list(frames[s])
        elif turn % 5 == 2:
            moves = compact(model, total)
        assert not set(f for f, _ in moves) & set(t for _, t in moves)
        for f, t in moves:
            for r in range(P):
                data[t * P + r] = data.get(f * P + r)
        held = [p for h in model.held for p in h.values()]
        assert sorted(held + list(model.free)) == list(range(total))
        for s in range(S):
            for k, page in model.held[s].items():
                for r in range(P):
                    pos = k * P + r
                    if max(0, model.A[s] - left) <= pos < model.A[s]:
                        assert data[page * P + r] == frames[s][pos]


def test_attention_model():
    """The softmax written out, one row at a time."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, 8, generator=g).double() for n in (3, 5, 5))
    seen = torch.tensor([[1, 0, 0, 0, 0], [1, 1, 0, 1, 0], [0, 0, 0, 0, 0]]).bool()
    k[4], v[2] = math.nan, math.inf
    out, tol = attend(q, k, v, seen, 0.7, torch.float32)
    assert torch.equal(out[0], v[0]) and (out[2] == 0).all() and torch.isfinite(tol).all()
    w = [math.exp(0.7 * float(q[1] @ k[j])) for j in (0, 1, 3)]
    torch.testing.assert_close(out[1], (w[0] * v[0] + w[1] * v[1] + w[2] * v[3]) / sum(w))


def test_rotation_model():
    """A rotation keeps lengths, and a query and a key turned alike meet by their distance alone."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 64, generator=g).double()
    inv = 10000.0 ** (-torch.arange(0, 64, 2).double() / 64)
    for mixed in (False, True):
        at = lambda p: norm_rotate(x[None], None, torch.tensor([p]), inv, 0.0, mixed)[0][0]  # noqa: E731
        torch.testing.assert_close(at(5).norm(dim=-1), x.norm(dim=-1))
        torch.testing.assert_close(at(5)[0] @ at(2)[1], at(1003)[0] @ at(1000)[1])


def test_pool_places_are_the_blocks():
    pool = torch.arange(2 * 3 * 4 * 96).view(2, 3, 4, 96).half()
    flat = torch.arange(pool.numel())
    at = pool_places(pool)
    blocks = flat.view(2, 3, 3, 4, 32)
    assert at[1, 2, 3, 70] == blocks[1, 2, 70 // 32, 3, 70 % 32]
    rows = np.array([[5, 1, 0]])
    kp, _, k, _ = fill_pages(rows, 4, 2, 96, [3], [6], torch.float16, torch.Generator().manual_seed(0))
    assert torch.equal(kp.view(-1)[pool_places(kp)[1, 1, 3]], k[0][0]) and torch.isnan(kp.view(-1)[pool_places(kp)[1, 1, 2]]).all()
    assert torch.equal(kp.view(-1)[pool_places(kp)[1, 0, 1]], k[0][2])


@pytest.mark.parametrize("args", [_lib.QkNormAppendArgs, _lib.ChunkAttnArgs, _lib.CrossAttnArgs, _lib.PageForkArgs, _lib.KvMovePagesArgs])
def test_packed_arguments_are_the_structure(args):
    """The bytes that a packer makes are the structure's, field by field; values out of a field's range are refused."""
    kinds = [kind for _, kind in _lib._layout(args)]
    values = [{"f": 0.5 + i, "Q": 2**63 + i}.get(kind, 100 + i) for i, kind in enumerate(kinds)]
    data = _lib.packer(args)(*values)
    a = args.from_buffer_copy(data)
    assert len(data) == ctypes.sizeof(args)

    def flat(s):
        for name, kind in s._fields_:
            x = getattr(s, name)
            yield from flat(x) if isinstance(x, ctypes.Structure) else (x,)

    assert list(flat(a)) == values
    for i, kind in enumerate(kinds):
        bad = list(values)
        bad[i] = 1e39 if kind == "f" else 2**64
        with pytest.raises(ValueError, match=args.__name__):
            _lib.packer(args)(*bad)
