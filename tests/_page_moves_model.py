"""Forks and compaction of a page pool, pair by pair and page by page, with a queue and lists."""

from tests._tables_model import RaggedPool


def fork(model: RaggedPool, src, dst):
    """The moves of a fork; `model` follows it."""
    slots, named, seen, pairs = range(len(model.A)), set(src), set(), []
    for s, d in zip(src, dst):
        if s in slots and d in slots and d not in named and d not in seen:
            pairs.append((s, d))
        seen.add(d)
    for _, d in pairs:
        model.free.extend(model.held[d][k] for k in sorted(model.held[d]))
    moves = []
    for s, d in pairs:
        model.held[d] = {k: model.free.popleft() for k in sorted(model.held[s])}
        model.A[d] = model.A[s]
        moves += [(model.held[s][k], model.held[d][k]) for k in sorted(model.held[s])]
    return moves


def compact(model: RaggedPool, total):
    """The moves of a compaction; `model` follows it."""
    live = sorted(p for held in model.held for p in held.values())
    n = len(live)
    moves = list(zip([p for p in live if p >= n], sorted(set(range(n)) - set(live))))
    to = dict(moves)
    model.held = [{k: to.get(p, p) for k, p in held.items()} for held in model.held]
    model.free.clear()
    model.free.extend(range(n, total))
    return moves
