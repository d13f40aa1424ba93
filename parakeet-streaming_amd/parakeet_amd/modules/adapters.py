"""Low-rank adapters of many customers beside one encoder.

An adapter of a projection ``y = x W^T`` adds ``scale (x A^T) B^T``, A [r, K], B [N, r].
:class:`EncoderAdapters` holds those of up to ``num_adapters`` customers for the
feed-forward and attention projections of every layer
(parakeet/modules/feedforward.py:20-26, attention.py:92,122); a batch's streams
name theirs by number and run together:

    adapters = EncoderAdapters(encoder, num_adapters=32, rank=16)
    adapters.load(3, {"layers.0.self_attn.qkv": (A, B), ...}, scale=alpha / r)
    ids = torch.tensor([3, -1, 0, 3], dtype=torch.int32, device=device)  # -1: none
    out, state = encoder(x, state, length=length, adapters=adapters.step(ids, x.shape[1]))

``EncoderStepGraph(..., adapters=adapters, adapter_ids=ids)`` records the step; the
streams' numbers are then read from ``ids`` at each replay.  The reference has no
adapters.

A load or clear is several launches on torch's current stream, into banks that steps read:
it runs on the steps' stream with no step launched or replayed in between, or is ordered
before them by events.  While steps of another thread go on, load into a number that
no stream has, and then give it to the streams.
"""

from __future__ import annotations

from collections.abc import Mapping
from dataclasses import dataclass

import torch
from torch import Tensor, nn
from torch.nn import functional as F

from .. import _lib, ops

TARGETS = (
    "feed_forward1.linear1",
    "feed_forward1.linear2",
    "self_attn.qkv",
    "self_attn.linear_out",
    "feed_forward2.linear1",
    "feed_forward2.linear2",
)


class EncoderAdapters:
    """Adapters 0 .. num_adapters - 1 of an encoder's projections, in the encoder's dtype
    on its device; zero (the shared weights alone) until loaded.  Ranks up to ``rank``,
    a multiple of 8."""

    def __init__(self, encoder: nn.Module, num_adapters: int, rank: int, targets=TARGETS):
        G, r = int(num_adapters), int(rank)
        if not 0 < G <= _lib.ADAPTER_MAX or r % 8 or not 0 < r <= _lib.ADAPTER_MAX_RANK:
            raise ValueError(f"need 0 < num_adapters <= {_lib.ADAPTER_MAX} and a rank that is a multiple of 8, at most "
                             f"{_lib.ADAPTER_MAX_RANK}; got {num_adapters}, {rank}")
        targets = tuple(targets)
        unknown = [t for t in targets if t not in TARGETS]
        if unknown:
            raise ValueError(f"no such projections: {unknown} (of {TARGETS})")
        self.num_adapters, self.rank = G, r
        self.banks: list[dict[str, ops.Adapters]] = []
        for layer in encoder.layers:
            bank = {}
            for name in targets:
                w = layer.get_submodule(name).weight
                n, k = w.shape
                bank[name] = ops.Adapters(
                    torch.zeros((G, r, k), dtype=w.dtype, device=w.device),
                    torch.zeros((G, n, r), dtype=w.dtype, device=w.device),
                    torch.zeros(G, dtype=torch.float32, device=w.device),
                )
            self.banks.append(bank)

    def _bank(self, name: str) -> ops.Adapters:
        head, _, rest = name.partition(".")
        number, _, target = rest.partition(".")
        if head == "layers" and number.isdigit() and int(number) < len(self.banks) and target in self.banks[int(number)]:
            return self.banks[int(number)][target]
        raise KeyError(f"no adapters are kept for {name!r}")

    def _check(self, i: int) -> int:
        if not 0 <= int(i) < self.num_adapters:
            raise IndexError(f"adapter {i} out of range [0, {self.num_adapters})")
        return int(i)

    @torch.no_grad()
    def load(self, i: int, weights: Mapping[str, tuple[Tensor, Tensor]], scale: float = 1.0) -> None:
        """Adapter ``i`` becomes ``weights``: {"layers.<n>.<target>": (A [r', K], B [N, r'])} with
        r' <= rank; projections that it does not name get none.  The values are copied
        into the banks, which recorded steps read, each entry written once."""
        i, scale = self._check(i), float(scale)
        parts = {}
        for name, (a, b) in weights.items():
            bank = self._bank(name)
            r, k, n = a.shape[0] if a.dim() == 2 else -1, bank.a.shape[2], bank.b.shape[1]
            if not 0 < r <= self.rank or tuple(a.shape) != (r, k) or tuple(b.shape) != (n, r):
                raise ValueError(f"{name}: need A [r, {k}] and B [{n}, r] with 0 < r <= {self.rank}, got {tuple(a.shape)} and {tuple(b.shape)}")
            parts[id(bank)] = a, b, r
        for layer in self.banks:
            for bank in layer.values():
                a, b, r = parts.get(id(bank), (None, None, 0))
                if r:
                    bank.a[i, :r].copy_(a)
                    bank.b[i, :, :r].copy_(b)
                if r < self.rank:
                    bank.a[i, r:].zero_()
                    bank.b[i, :, r:].zero_()
                bank.scale[i] = scale if r else 0.0

    @torch.no_grad()
    def clear(self, i: int) -> None:
        """Adapter ``i`` adds nothing."""
        i = self._check(i)
        for layer in self.banks:
            for bank in layer.values():
                bank.a[i].zero_()
                bank.b[i].zero_()
                bank.scale[i] = 0.0

    def step(self, ids: Tensor, frames: int) -> "StepAdapters":
        """The adapters of one step's batch: stream b's ``frames`` rows use ``ids[b]``
        (int32 [B] on the device; a number outside the bank is no adapter)."""
        return StepAdapters(self, ops.adapter_plan(ids, frames, num_adapters=self.num_adapters))


@dataclass
class StepAdapters:
    """What the layers of one step read: the banks and the batch's plan."""

    adapters: EncoderAdapters
    plan: ops.AdapterPlan

    def linear(self, layer: int, name: str, m: nn.Module, x: Tensor, silu: bool = False) -> Tensor:
        """``m(x)`` of a layer's projection with the streams' adapters beside it, and SiLU."""
        bank = self.adapters.banks[layer].get(name)
        if bank is None:
            y = ops.module_linear(x, m)
            return F.silu(y) if silu else y
        if not ops.plain_module(m, nn.Linear):
            raise NotImplementedError(f"adapters beside a replaced or hooked {name}")
        return ops.adapter_linear(x, m.weight, m.bias, bank, self.plan, silu=silu)

    def feed_forward(self, layer: int, name: str, ff: nn.Module, x: Tensor) -> Tensor:
        """A feed-forward block (feedforward.py:20-26)."""
        if not ff._fused():
            raise NotImplementedError(f"adapters beside a {name} with active dropout, hooks or replaced parts")
        h = self.linear(layer, name + ".linear1", ff.linear1, x, silu=True)
        return self.linear(layer, name + ".linear2", ff.linear2, h)


__all__ = ["EncoderAdapters", "StepAdapters", "TARGETS"]
