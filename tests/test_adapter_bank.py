"""Loading adapters into the banks that steps read."""

import torch
from torch import nn
from torch.utils._python_dispatch import TorchDispatchMode

from parakeet_amd.modules.adapters import TARGETS, EncoderAdapters


class _Writes(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(func.overloadpacket.__name__)
        return func(*args, **(kwargs or {}))


class _Layer(nn.Module):
    def __init__(self, d):
        super().__init__()
        for name in TARGETS:
            block, proj = name.split(".")
            if not hasattr(self, block):
                setattr(self, block, nn.Module())
            n, k = {"linear1": (4 * d, d), "linear2": (d, 4 * d), "qkv": (3 * d, d), "linear_out": (d, d)}[proj]
            setattr(getattr(self, block), proj, nn.Linear(k, n))


def _bank(layers=2, d=64, G=3, rank=16):
    enc = nn.Module()
    enc.layers = nn.ModuleList(_Layer(d) for _ in range(layers))
    ad = EncoderAdapters(enc, G, rank)

    def weights(r, names, seed):
        g = torch.Generator().manual_seed(seed)
        w = {}
        for layer in range(layers):
            for name in names:
                b = ad.banks[layer][name]
                w[f"layers.{layer}.{name}"] = (torch.randn(r, b.a.shape[2], generator=g), torch.randn(b.b.shape[1], r, generator=g))
        return w

    return ad, weights


def test_a_load_writes_each_entry_once():
    """An adapter in use is never cleared first: between the two a step would have none."""
    ad, weights = _bank()
    ad.load(1, weights(16, TARGETS, 0), 2.0)
    with _Writes() as w:
        ad.load(1, weights(16, TARGETS, 1), 0.5)
    assert "zero_" not in w.seen and w.seen.count("copy_") >= 2 * 2 * len(TARGETS)


def test_a_load_leaves_nothing_of_the_adapter_before():
    ad, weights = _bank()
    ad.load(0, weights(16, TARGETS, 3), 3.0)
    ad.load(2, weights(8, TARGETS, 4), 4.0)
    before = [(b.a.clone(), b.b.clone(), b.scale.clone()) for layer in ad.banks for b in layer.values()]
    new = weights(8, TARGETS[1:4], 5)
    ad.load(0, new, 0.25)
    for layer in range(2):
        for j, name in enumerate(TARGETS):
            bank, (a, b, s) = ad.banks[layer][name], before[layer * len(TARGETS) + j]
            assert torch.equal(bank.a[1:], a[1:]) and torch.equal(bank.b[1:], b[1:]) and torch.equal(bank.scale[1:], s[1:])
            if name in TARGETS[1:4]:
                x, y = new[f"layers.{layer}.{name}"]
                assert torch.equal(bank.a[0, :8], x) and torch.equal(bank.b[0, :, :8], y) and bank.scale[0] == 0.25
                assert not bank.a[0, 8:].any() and not bank.b[0, :, 8:].any()
            else:
                assert not bank.a[0].any() and not bank.b[0].any() and bank.scale[0] == 0
    ad.clear(0)
    assert all(not b.a[0].any() and not b.b[0].any() and b.scale[0] == 0 for layer in ad.banks for b in layer.values())
