"""Performance cases of the operators that a text decoder needs to read this framework's
encoder and to keep its own tokens on the same pages.

* ``project``: queries and keys normed head by head and rotated to their positions, keys
  and values into their pages in the same pass (``ops.qk_norm_append``);
* ``chunk``: new tokens of each stream attend over its paged cache, grouped heads
  (``ops.chunk_attn``);
* ``cross``: tokens attend to the encoder's states of another length (``ops.cross_attn``);
* ``fork``: streams forked page by page (``ops.page_fork``, ``ops.kv_move_pages``), and the live
  pages moved together afterwards where ``compact`` is set (``ops.page_compact``).

Widths are those of the two models served here (512 columns in heads of 64, 1024 in heads
of 128) and a decoder of 2048 columns, from one stream to hundreds.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "parakeet-streaming_amd")
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
DEV = "cuda"
EPS = 1e-6


# ---------------------------------------------------------------------------
# cases


def _project(streams, tokens, ragged, heads, kv_heads, hd, rot, interleaved, page, far, dtype):
    return {"kind": "project", "streams": streams, "tokens": tokens, "ragged": ragged, "heads": heads, "kv_heads": kv_heads, "hd": hd,
            "rot": rot, "interleaved": interleaved, "page": page, "far": far, "dtype": dtype}


def _chunk(streams, tokens, ragged, history, left, heads, kv_heads, hd, page, dtype):
    return {"kind": "chunk", "streams": streams, "tokens": tokens, "ragged": ragged, "history": history, "left": left, "heads": heads,
            "kv_heads": kv_heads, "hd": hd, "page": page, "dtype": dtype}


def _cross(streams, tokens, states, ragged, heads, kv_heads, hd, dtype):
    return {"kind": "cross", "streams": streams, "tokens": tokens, "states": states, "ragged": ragged, "heads": heads, "kv_heads": kv_heads,
            "hd": hd, "dtype": dtype}


def _fork(pairs, slots, compact, layers, d, left, tokens, page, dtype):
    return {"kind": "fork", "pairs": pairs, "slots": slots, "compact": compact, "layers": layers, "d": d, "left": left, "tokens": tokens,
            "page": page, "dtype": dtype}


def listed():
    return [
        # one token of each of 8 streams of a small decoder: latency
        dict(_project(8, 1, False, 8, 8, 64, 64, False, 16, 4000, "fp16"), name="project_8"),
        # the prompts of 61 streams, some shorter, eight query heads to a key head
        dict(_project(61, 256, True, 16, 2, 128, 128, False, 16, 100000, "bf16"), name="project_prompt_61"),
        # one token of each of 8 streams over short utterances: latency
        dict(_chunk(8, 1, False, 190, 0, 8, 8, 64, 16, "fp16"), name="chunk_8"),
        # one stream far into a long recording
        dict(_chunk(1, 1, False, 61443, 0, 16, 2, 128, 16, "bf16"), name="chunk_long_1"),
        # a serving batch, caches from empty to 4096 tokens
        dict(_chunk(128, 1, True, 4095, 0, 16, 4, 128, 16, "bf16"), name="chunk_128"),
        # up to 5 drafted tokens of 60 streams, a window of 512 tokens
        dict(_chunk(60, 5, True, 9000, 511, 8, 8, 64, 16, "fp16"), name="chunk_draft_60"),
        # prompts of 512 tokens behind 3500 earlier ones
        dict(_chunk(4, 512, False, 3500, 0, 16, 4, 128, 32, "bf16"), name="chunk_prompt_4"),
        # one token of 8 streams to 30 seconds of encoder states: latency
        dict(_cross(8, 1, 376, False, 8, 8, 64, "fp16"), name="cross_8"),
        # 4 hypotheses of 60 streams to recordings of up to two minutes
        dict(_cross(60, 4, 1500, True, 8, 8, 128, "bf16"), name="cross_beams_60"),
        # whole texts scored in an fp32 deployment of the small model
        dict(_cross(8, 197, 751, True, 8, 8, 64, "fp32"), name="cross_fp32_8"),
        # 4 streams of the small model forked, 17 layers
        dict(_fork(4, 32, False, 17, 512, 70, 2, 16, "fp16"), name="fork_4"),
        # 48 of 230 streams of the large model end and start again as forks of others; the pool is compacted
        dict(_fork(48, 230, True, 24, 1024, 70, 14, 16, "bf16"), name="compact_48"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["project", "chunk", "chunk", "cross", "cross", "fork"])
    dtype = rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"])
    hd = rng.choice([64, 128])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 8]) if kv <= 2 else kv * rng.choice([1, 1, 2, 4])
    page = rng.choice([8, 16, 16, 32])
    if kind == "project":
        tokens = rng.choice([1, 1, 2, 5, _log_int(rng, 6, 300)])
        streams = _log_int(rng, 1, max(1, 12000 * 20 * 128 // (tokens * (heads + 2 * kv) * hd) // (2 if dtype == "fp32" else 1)))
        return _project(min(streams, 4000), tokens, rng.random() < 0.5, heads, kv, hd, rng.choice([hd, hd, hd // 2]), rng.random() < 0.3, page,
                        rng.choice([1000, 100000, 1000000]), dtype)
    slow = 8 if dtype == "fp32" else 1
    if kind == "chunk":
        tokens = rng.choice([1, 1, 1, 3, 5, _log_int(rng, 8, 512)])
        history = _log_int(rng, 1, 40000 if tokens == 1 else 6000)
        left = 0 if rng.random() < 0.7 else min(history, _log_int(rng, 32, 2048))
        seen = (left or history) + tokens
        most = min(1.3e8 / slow / (seen * kv * hd), 5e10 / slow / (4 * seen * tokens * heads * hd))
        return _chunk(_log_int(rng, 1, max(1, min(256, int(most)))), tokens, rng.random() < 0.6, history, left, heads, kv, hd, page, dtype)
    if kind == "cross":
        tokens = rng.choice([1, 1, 4, 5, _log_int(rng, 8, 448)])
        states = _log_int(rng, 1, 4000)
        most = min(4.5e7 / slow / (states * kv * hd), 5e10 / slow / (4 * states * tokens * heads * hd))
        return _cross(_log_int(rng, 1, max(1, min(256, int(most)))), tokens, states, rng.random() < 0.6, heads, kv, hd, dtype)
    d, layers = rng.choice([(512, 17), (512, 4), (1024, 24), (1024, 8)])
    left = rng.choice([70, 70, 200, 600])
    slots = _log_int(rng, 4, max(4, 230 * 24 * 1024 * 80 // (layers * d * (left + 10) * (2 if dtype == "fp32" else 1))))
    slots = min(slots, 1000)
    return _fork(rng.randint(1, max(1, slots // 5)), slots, rng.random() < 0.5, layers, d, left, rng.choice([1, 2, 14]), page, dtype)


# ---------------------------------------------------------------------------
# inputs


def _entries(left, tokens, page):
    """Ring entries a window of left + tokens frames needs."""
    return (left + tokens + page - 2) // page + 1


def _column_block(d, dtype):
    return math.gcd(d, 64 // SIZE[dtype])


def _pages_of(c):
    """(left, ring entries) of a chunk case's cache."""
    left = c["left"] or c["history"]
    return left, _entries(left, c["tokens"], c["page"])


def _held(A, window, page, M):
    """[S, M] whether a ring entry of a slot of A frames holds a page."""
    lo, hi = np.maximum(A - window, 0) // page, (A + page - 1) // page
    r = np.arange(M)[None, :]
    return (lo[:, None] + (r - lo[:, None]) % M) < hi[:, None]


def _up(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def prepare(case, seed):
    c = case
    rng = np.random.default_rng(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    rnd = lambda *s, std=1.0: (torch.randn(s, generator=g, device=DEV) * std).to(dt)  # noqa: E731
    if c["kind"] == "project":
        n, T, P, Hq, Hkv, hd = (c[k] for k in ("streams", "tokens", "page", "heads", "kv_heads", "hd"))
        # each stream's new tokens behind A earlier ones, in pages of its own
        A = rng.integers(0, c["far"], n)
        per = (T + 2 * P - 2) // P
        pages = rng.permutation(n * per).reshape(n, per)
        pos = A[:, None] % P + np.arange(T)[None, :]
        slot = np.take_along_axis(pages, pos // P, 1) * P + pos % P
        if c["ragged"]:
            slot = np.where(np.arange(T)[None, :] < rng.integers(0, T + 1, n)[:, None], slot, -1)
        x = rnd(n, T, (Hq + 2 * Hkv) * hd, std=2.0)  # q | k | v as the projection leaves them
        rows = np.concatenate([A[:, None], pages], 1).astype(np.int32)
        inv = 10000.0 ** (-np.arange(0, c["rot"], 2, dtype=np.float64) / c["rot"])
        return {"case": c, "query": x[..., : Hq * hd], "key": x[..., Hq * hd : (Hq + Hkv) * hd], "value": x[..., (Hq + Hkv) * hd :],
                "k_pool": rnd(1, n * per, P, Hkv * hd), "v_pool": rnd(1, n * per, P, Hkv * hd), "slot_map": _up(slot.astype(np.int32)), "rows": _up(rows),
                "q_weight": (1 + rnd(hd, std=0.2)).to(dt), "k_weight": (1 + rnd(hd, std=0.2)).to(dt), "inv_freq": _up(inv)}
    if c["kind"] == "chunk":
        n, T, P, Hq, Hkv, hd = (c[k] for k in ("streams", "tokens", "page", "heads", "kv_heads", "hd"))
        left, M = _pages_of(c)
        # history: the most tokens before the new ones; ragged batches have any number up to it and some streams few new tokens
        A = np.full(n, c["history"])
        new = np.full(n, T)
        if c["ragged"]:
            A = rng.integers(0, c["history"] + 1, n)
            new = rng.integers(1, T + 1, n)
        held = _held(A + new, left + T, P, M)
        pages = rng.permutation(n * M).reshape(n, M)
        rows = np.concatenate([A[:, None], np.where(held, pages, -1)], 1).astype(np.int32)
        return {"case": c, "query": rnd(n, T, Hq * hd), "k_pool": rnd(1, n * M, P, Hkv * hd), "v_pool": rnd(1, n * M, P, Hkv * hd), "rows": _up(rows),
                "lengths": _up(new.astype(np.int32))}
    if c["kind"] == "cross":
        n, T, S, Hq, Hkv, hd = (c[k] for k in ("streams", "tokens", "states", "heads", "kv_heads", "hd"))
        lens = rng.integers(0, S + 1, n) if c["ragged"] else np.full(n, S)
        kv = rnd(n, S, 2 * Hkv * hd)  # k | v as the projection of the states leaves them
        return {"case": c, "query": rnd(n, T, Hq * hd), "key": kv[..., : Hkv * hd], "value": kv[..., Hkv * hd :], "lengths": _up(lens.astype(np.int32))}
    # fork: every slot has a stream, the live pages are the pool's first, in no order
    S, P, n, W = c["slots"], c["page"], c["pairs"], c["left"] + c["tokens"]
    M = _entries(c["left"], c["tokens"], P)
    A = rng.integers(1, 6 * W, S)
    held = _held(A, W, P, M)
    live = int(held.sum())
    ring = np.full((S, M), -1, dtype=np.int32)
    ring[held] = rng.permutation(live)
    queue = np.zeros(S * M, dtype=np.int32)
    first = int(rng.integers(0, S * M))
    queue[(first + np.arange(S * M - live)) % (S * M)] = live + rng.permutation(S * M - live)
    slots = rng.permutation(S)
    src = rng.choice(slots[n:], n)  # a stream may be forked more than once
    pool = lambda: torch.empty((c["layers"], S * M, P, c["d"]), dtype=dt, device=DEV).normal_(generator=g)  # noqa: E731
    return {"case": c, "queue": _up(queue), "head": _up(np.array([first, S * M - live], dtype=np.int32)), "appended": _up(A.astype(np.int64)), "ring": _up(ring),
            "src": _up(src.astype(np.int32)), "dst": _up(slots[:n].astype(np.int32)), "k_pool": pool(), "v_pool": pool()}


# ---------------------------------------------------------------------------
# plain forms


def _heads(x, hd):
    """[B, T, H hd] -> fp32 [B, H, T, hd]."""
    B, T, D = x.shape
    return x.float().view(B, T, D // hd, hd).transpose(1, 2)


def _blocks(pool):
    """A page pool by (layer, page, column block of 64 bytes, row, column)."""
    ly, pages, P, D = pool.shape
    cb = math.gcd(D, 64 // pool.element_size())
    return pool.view(ly, pages, D // cb, P, cb)


def _plain_norm_rotate(x, weight, hd, rot, interleaved, cos, sin):
    """x [B, T, H hd], cos and sin [B, T, 1, rot / 2]."""
    B, T, D = x.shape
    y = x.float().view(B, T, D // hd, hd)
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    r, rest = y[..., :rot], y[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., : rot // 2], r[..., rot // 2 :])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([r, rest], -1).view(B, T, D).to(x.dtype)


def _plain_project(s):
    c = s["case"]
    P, hd, T = c["page"], c["hd"], c["tokens"]
    pos = s["rows"][:, :1].double() + torch.arange(T, device=DEV)
    angle = (pos[..., None] * s["inv_freq"])[:, :, None, :]
    turn = (hd, c["rot"], c["interleaved"], torch.cos(angle).float(), torch.sin(angle).float())
    q = _plain_norm_rotate(s["query"], s["q_weight"], *turn)
    k = _plain_norm_rotate(s["key"], s["k_weight"], *turn)
    slot = s["slot_map"].reshape(-1).long()
    keep = slot >= 0
    slot = slot[keep]
    for pool, x in ((s["k_pool"], k), (s["v_pool"], s["value"])):
        b = _blocks(pool)[0]
        b[slot // P, :, slot % P] = x.reshape(-1, x.shape[-1])[keep].view(-1, b.shape[1], b.shape[3])
    return q


def _plain_attention(q, k, v, seen):
    """q [B, Hkv, G, T, hd], k and v [B, Hkv, L, hd] in fp32, seen bool [B, 1, 1, T, L]; a query that sees nothing gets zeros."""
    B, Hkv, G, T, hd = q.shape
    x = torch.matmul(q.reshape(B, Hkv, G * T, hd), k.transpose(2, 3).contiguous()).view(B, Hkv, G, T, -1) * hd**-0.5
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
    e = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return torch.matmul(e.view(B, Hkv, G * T, -1), v).view(B, Hkv * G, T, hd).transpose(1, 2).reshape(B, T, -1)


def _plain_chunk(s):
    c = s["case"]
    P, hd, T, Hkv = c["page"], c["hd"], c["tokens"], c["kv_heads"]
    left, M = _pages_of(c)
    A, ring = s["rows"][:, 0].long(), s["rows"][:, 1:].long()
    new = s["lengths"].long().clamp(0, T)
    # absolute position of each row of each ring entry: the newest page of its residue
    last = (A + new - 1).clamp(min=0) // P
    page = last[:, None] - (last[:, None] - torch.arange(M, device=DEV)) % M
    pos = (page[:, :, None] * P + torch.arange(P, device=DEV)).view(-1, 1, M * P)
    there = ((ring >= 0) & (page >= 0))[:, :, None].expand(-1, -1, P).reshape(-1, 1, M * P) & (pos < (A + new)[:, None, None])
    at = A[:, None, None] + torch.arange(T, device=DEV)[None, :, None]
    seen = there & (pos <= at) & (pos >= at - left) & (at < (A + new)[:, None, None])
    dense = lambda pool: _blocks(pool)[0][ring.clamp(min=0)].transpose(2, 3).reshape(len(A), M * P, -1)  # noqa: E731
    k, v = _heads(dense(s["k_pool"]), hd), _heads(dense(s["v_pool"]), hd)
    v = torch.where(there[:, :, :, None], v, 0.0)
    q = _heads(s["query"], hd).unflatten(1, (Hkv, -1))
    return _plain_attention(q, k, v, seen[:, None, None]).to(s["query"].dtype)


def _plain_cross(s):
    c = s["case"]
    k, v = _heads(s["key"], c["hd"]), _heads(s["value"], c["hd"])
    there = torch.arange(c["states"], device=DEV)[None, :] < s["lengths"][:, None]
    v = torch.where(there[:, None, :, None], v, 0.0)
    q = _heads(s["query"], c["hd"]).unflatten(1, (c["kv_heads"], -1))
    return _plain_attention(q, k, v, there[:, None, None, None, :]).to(s["query"].dtype)


def _plain_move(s, pairs, count):
    pairs = pairs[:count].long()
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, pairs[:, 1]] = pool[:, pairs[:, 0]]


def _plain_fork(s):
    c = s["case"]
    P, W = c["page"], c["left"] + c["tokens"]
    queue, head, A, ring = s["queue"], s["head"].long(), s["appended"], s["ring"]
    total, M = queue.numel(), ring.shape[1]
    src, dst = s["src"].long(), s["dst"].long()
    r = torch.arange(M, device=DEV)
    # the pages of the slots that are replaced to the back of the queue, oldest first
    lo, hi = (A[dst] - W).clamp(min=0) // P, (A[dst] + P - 1) // P
    k = (r + lo[:, None]) % M
    had = r < (hi - lo)[:, None]
    back = torch.cumsum(hi - lo, 0) - (hi - lo)
    queue[((head[0] + head[1] + back[:, None] + r) % total)[had]] = ring[dst[:, None], k][had]
    # as many from its front as the forked ones hold
    lo2, hi2 = (A[src] - W).clamp(min=0) // P, (A[src] + P - 1) // P
    k = (r + lo2[:, None]) % M
    takes = r < (hi2 - lo2)[:, None]
    at = torch.cumsum(hi2 - lo2, 0) - (hi2 - lo2)
    got = queue[(head[0] + at[:, None] + r) % total]
    pairs = torch.stack([ring[src[:, None], k][takes], got[takes]], 1)
    fresh = torch.full((len(dst), M), -1, dtype=torch.int32, device=DEV)
    fresh.scatter_(1, k, torch.where(takes, got, -1))
    ring[dst] = fresh
    A[dst] = A[src]
    given, taken = (hi - lo).sum(), (hi2 - lo2).sum()
    s["head"].copy_(torch.stack([(head[0] + taken) % total, head[1] + given - taken]))
    _plain_move(s, pairs, len(pairs))


def _plain_compact(s):
    queue, ring = s["queue"], s["ring"]
    total = queue.numel()
    pages = torch.arange(total, device=DEV)
    live = torch.zeros(total, dtype=torch.bool, device=DEV)
    live[ring[ring >= 0].long()] = True
    n = live.sum()
    frm, to = torch.nonzero(live & (pages >= n))[:, 0], torch.nonzero(~live & (pages < n))[:, 0]
    new = pages.clone()
    new[frm] = to
    ring.copy_(torch.where(ring >= 0, new[ring.clamp(min=0).long()].to(torch.int32), ring))
    queue.copy_(torch.where(pages < total - n, n + pages, queue))
    s["head"].copy_(torch.stack([torch.zeros_like(n), total - n]))
    _plain_move(s, torch.stack([frm, to], 1), len(frm))


# ---------------------------------------------------------------------------
# one pass


def _ops():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from parakeet_amd import ops

    return ops


def _own_fork(s):
    ops, c = _ops(), s["case"]
    st = ops.PageState(s["queue"], s["head"], s["appended"], s["ring"], page_size=c["page"], left=c["left"], chunk=c["tokens"])
    ops.kv_move_pages(s["k_pool"], s["v_pool"], ops.page_fork(st, s["src"], s["dst"]))
    if c["compact"]:
        ops.kv_move_pages(s["k_pool"], s["v_pool"], ops.page_compact(st))


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "project":
        if own:
            ops = _ops()
            pages = ops.PagedKV(s["k_pool"], s["v_pool"], s["rows"], s["rows"].shape[1] - 1)
            q = ops.qk_norm_append(s["query"], s["key"], s["value"], pages, 0, s["slot_map"], num_heads=c["heads"], q_weight=s["q_weight"],
                                   k_weight=s["k_weight"], inv_freq=s["inv_freq"], eps=EPS, interleaved=c["interleaved"])
        else:
            q = _plain_project(s)
        return {"query": q, "k": s["k_pool"], "v": s["v_pool"]}
    if kind == "chunk":
        if own:
            ops = _ops()
            pages = ops.PagedKV(s["k_pool"], s["v_pool"], s["rows"], s["rows"].shape[1] - 1)
            return ops.chunk_attn(s["query"], pages, 0, num_heads=c["heads"], lengths=s["lengths"], left=_pages_of(c)[0])
        return _plain_chunk(s)
    if kind == "cross":
        if own:
            return _ops().cross_attn(s["query"], s["key"], s["value"], num_heads=c["heads"], lengths=s["lengths"])
        return _plain_cross(s)
    if own:
        _own_fork(s)
    else:
        _plain_fork(s)
        if c["compact"]:
            _plain_compact(s)
    return {"queue": s["queue"], "head": s["head"], "appended": s["appended"], "ring": s["ring"], "k": s["k_pool"], "v": s["v_pool"]}


# ---------------------------------------------------------------------------
# what a pass cannot do without


def _pairs_seen(c):
    """(keys that some query of a stream sees, query-key pairs of a head), a stream in the mean."""
    T, left = c["tokens"], c["left"] or c["history"]
    hist = c["history"] / 2 if c["ragged"] else c["history"]
    new = (T + 1) / 2 if c["ragged"] else T
    return min(hist, left) + new, new * min(hist + (new + 1) / 2, left + 1)


def work(case):
    c = case
    e = SIZE[c["dtype"]]
    if c["kind"] == "project":
        tokens = c["streams"] * c["tokens"]
        written = tokens / 2 if c["ragged"] else tokens  # K and V of tokens past a stream's are neither read nor written
        return {"bytes": e * c["hd"] * 2 * (tokens * c["heads"] + written * 2 * c["kv_heads"]) + 4 * tokens, "flops": 0}
    if c["kind"] == "chunk":
        keys, pairs = _pairs_seen(c)
        n = c["streams"]
        return {"bytes": e * c["hd"] * 2 * n * (keys * c["kv_heads"] + c["tokens"] * c["heads"]), "flops": 4.0 * c["hd"] * n * pairs * c["heads"]}
    if c["kind"] == "cross":
        keys = c["states"] / 2 if c["ragged"] else c["states"]
        n, T = c["streams"], c["tokens"]
        return {"bytes": e * c["hd"] * 2 * n * (keys * c["kv_heads"] + T * c["heads"]), "flops": 4.0 * c["hd"] * n * T * keys * c["heads"]}
    # pages of a stream in the mean, read and written in K and V of every layer, twice with the compaction
    per = (c["left"] + c["tokens"]) / c["page"]
    return {"bytes": (2 if c["compact"] else 1) * c["pairs"] * per * c["page"] * c["d"] * e * 4 * c["layers"], "flops": 0}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits


def _cells(slot, page, d, dtype):
    """[n, d] element offsets, in a layer's pool, of the columns of the frames at places ``slot``."""
    cb = _column_block(d, dtype)
    col = torch.arange(d, device=DEV)
    slot = torch.as_tensor(slot, device=DEV).long()[:, None]
    return slot // page * (page * d) + col // cb * (page * cb) + slot % page * cb + col % cb


def _exact_project(s):
    c = s["case"]
    hd, rot, T = c["hd"], c["rot"], c["tokens"]
    pos = s["rows"][:, 0].double()[:, None] + torch.arange(T, device=DEV, dtype=torch.float64)[None]
    angle = pos[:, :, None] * s["inv_freq"]
    phase = torch.polar(torch.ones_like(angle), angle)  # e^(i pos f)
    out = []
    for x, w in ((s["query"], s["q_weight"]), (s["key"], s["k_weight"])):
        y = x.double().unflatten(-1, (-1, hd))
        y = y / (y.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
        i = torch.arange(rot // 2, device=DEV)
        a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + rot // 2)
        z = torch.complex(y[..., a], y[..., b]) * phase[:, :, None]
        y[..., a], y[..., b] = z.real, z.imag
        out.append(y.flatten(-2))
    slot = s["slot_map"].reshape(-1)
    at = (slot >= 0).nonzero()[:, 0]
    cells = _cells(slot[at], c["page"], c["kv_heads"] * hd, c["dtype"])
    pools = []
    for pool, x in ((s["k_pool"], out[1]), (s["v_pool"], s["value"].double())):
        p = pool.double()
        p.view(-1)[cells] = x.reshape(-1, x.shape[-1])[at]
        pools.append(p)
    return {"query": out[0], "k": pools[0], "v": pools[1]}


def _exact_rows(q, k, v, seen):
    """q [H, T, hd] of one group of heads, k and v [L, hd], seen [T, L], all in 64 bits."""
    x = torch.matmul(q, k.t().contiguous()) / math.sqrt(k.shape[1])
    x = x.masked_fill(~seen, -math.inf)
    p = torch.softmax(x, -1)
    return torch.matmul(torch.where(seen.any(-1)[:, None], p, 0.0), v)


def _exact_chunk(s):
    c = s["case"]
    P, hd, T, Hkv = c["page"], c["hd"], c["tokens"], c["kv_heads"]
    left, M = _pages_of(c)
    rows, new = s["rows"].cpu().numpy(), s["lengths"].cpu().numpy()
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
    for b in range(c["streams"]):
        A, n = int(rows[b, 0]), int(new[b])
        pos = np.arange(max(0, A - left), A + n)
        cells = _cells(rows[b, 1 + pos // P % M].astype(np.int64) * P + pos % P, P, Hkv * hd, c["dtype"])
        k, v = (s[p][0].reshape(-1)[cells].double().view(-1, Hkv, hd) for p in ("k_pool", "v_pool"))
        q = s["query"][b, :n].double().view(n, Hkv, -1, hd)
        j, i = torch.from_numpy(pos).to(DEV)[None, :], A + torch.arange(n, device=DEV)[:, None]
        seen = (j <= i) & (i - j <= left)
        for h in range(Hkv):
            o = _exact_rows(q[:, h].transpose(0, 1).contiguous(), k[:, h].contiguous(), v[:, h].contiguous(), seen)
            out[b, :n].view(n, Hkv, -1, hd)[:, h] = o.transpose(0, 1)
    return out


def _exact_cross(s):
    c = s["case"]
    hd, Hkv = c["hd"], c["kv_heads"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        k, v = (s[p][b, :n].double().view(n, Hkv, hd) for p in ("key", "value"))
        q = s["query"][b].double().view(c["tokens"], Hkv, -1, hd)
        for h in range(Hkv):
            seen = torch.ones(c["tokens"], n, dtype=torch.bool, device=DEV)
            o = _exact_rows(q[:, h].transpose(0, 1).contiguous(), k[:, h].contiguous(), v[:, h].contiguous(), seen)
            out[b].view(c["tokens"], Hkv, -1, hd)[:, h] = o.transpose(0, 1)
    return out


def _exact_fork(s):
    """The pool stream by stream, with a queue and lists."""
    c = s["case"]
    P, W = c["page"], c["left"] + c["tokens"]
    queue, head, A, ring = (s[k].cpu().numpy().copy() for k in ("queue", "head", "appended", "ring"))
    total, M = len(queue), ring.shape[1]
    first, count = int(head[0]), int(head[1])
    logical = lambda a: range(max(0, a - W) // P, (a + P - 1) // P)  # noqa: E731
    k, v = s["k_pool"].clone(), s["v_pool"].clone()

    def move(moves):
        f, t = (torch.tensor(x, device=DEV, dtype=torch.int64) for x in zip(*moves))
        for pool in (k, v):
            pool[:, t] = pool[:, f]

    src, dst = s["src"].tolist(), s["dst"].tolist()
    for d in dst:
        for p in logical(int(A[d])):
            queue[(first + count) % total], ring[d, p % M] = ring[d, p % M], -1
            count += 1
    moves = []
    for a, d in zip(src, dst):
        for p in logical(int(A[a])):
            ring[d, p % M] = queue[first]
            moves.append((int(ring[a, p % M]), int(queue[first])))
            first, count = (first + 1) % total, count - 1
        A[d] = A[a]
    move(moves)
    if c["compact"]:
        live = sorted(int(p) for p in ring.reshape(-1) if p >= 0)
        n = len(live)
        holes = sorted(set(range(n)) - set(live))
        moves = list(zip([p for p in live if p >= n], holes))
        to = dict(moves)
        ring = np.vectorize(lambda p: to.get(int(p), int(p)), otypes=[np.int32])(ring)
        queue[: total - n] = np.arange(n, total)
        first, count = 0, total - n
        if moves:
            move(moves)
    return {"queue": queue, "head": np.array([first, count], dtype=np.int32), "appended": A, "ring": ring, "k": k.double(), "v": v.double()}


def exact(case, seed):
    s = prepare(case, seed)
    return {"project": _exact_project, "chunk": _exact_chunk, "cross": _exact_cross, "fork": _exact_fork}[case["kind"]](s)
