"""The per-request tables and weights of a step together, as a serving loop uses them:
the encoder on pages kept in device memory, with each stream's adapters, eager and
recorded; and a ragged attention step from the operators themselves."""

import copy
import math

import numpy as np
import pytest
import torch

from oracle import attention as oa
from parakeet_amd import ops, synth
from parakeet_amd.modules.adapters import TARGETS, EncoderAdapters
from parakeet_amd.modules.encoder import ConformerEncoder, EncoderStepGraph
from parakeet_amd.pool import DevicePagePool

from _dense_encoder import init_attention

pytestmark = pytest.mark.gpu

LEFT, RIGHT, D, H, LY, P = 10, 1, 128, 2, 2, 4
T = RIGHT + 1


def _encoder(cuda, dtype, left=LEFT, right=RIGHT):
    torch.manual_seed(5)
    enc = ConformerEncoder(
        feat_in=80, hidden_size=D, ff_expansion_factor=2, num_layers=LY, num_heads=H, subsampling_factor=8, pos_emb_max_len=64,
        conv_kernel_size=9, att_context_size=[left, right], subsampling_conv_channels=32, use_bias=False, page_size=P,
    )
    for layer in enc.layers:
        init_attention(layer.self_attn, D, seed=20 + layer.layer_idx)
    return enc.to(cuda).to(dtype).eval().requires_grad_(False)


def _same(a, b):
    assert torch.equal(a.processed_frames, b.processed_frames) and torch.equal(a.cache_lengths, b.cache_lengths)
    assert torch.equal(a.cache.conv_frames, b.cache.conv_frames)
    for layer in range(LY):
        for x, y in zip(a.cache.window(layer), b.cache.window(layer)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_encoder_on_device_pages(cuda, dtype):
    """The same bits as on host pages, eager and recorded, with slots reset between steps."""
    enc = _encoder(cuda, dtype)
    B = 5
    length = torch.full((B,), T, dtype=torch.int64, device=cuda)
    host, eager, replay = (enc.init_streaming_state(batch_size=B, device=cuda, dtype=dtype, device_pages=d) for d in (False, True, True))
    graph = EncoderStepGraph(enc, replay, length)
    g = torch.Generator().manual_seed(6)
    with torch.no_grad():
        for step in range(14):
            x = torch.randn(B, T, D, generator=g).to(dtype).to(cuda)
            want, _ = enc(x, host, length=length)
            assert torch.equal(enc(x, eager, length=length)[0], want)
            assert torch.equal(graph(x), want), step
            _same(host, eager)
            _same(host, replay)
            if step % 4 == 3:
                for state in (host, eager, replay):
                    for s in (step % B, (step + 2) % B):
                        state.processed_frames[s : s + 1].zero_()
                        state.cache_lengths[s : s + 1].zero_()
                        state.cache.reset_slot(s)
    assert host.cache.pool.free_list().tolist() == eager.cache.pool.free_list().tolist() == replay.cache.pool.free_list().tolist()


def test_batches_of_changing_slots_on_device_pages(cuda):
    enc = _encoder(cuda, torch.float16)
    S = 7
    states = [enc.init_streaming_state(batch_size=S, device=cuda, dtype=torch.float16, device_pages=d) for d in (False, True)]
    rng = np.random.default_rng(3)
    g = torch.Generator().manual_seed(7)
    with torch.no_grad():
        for step in range(16):
            slots = rng.permutation(S)[: rng.integers(1, S + 1)].tolist()
            at = torch.tensor(slots, device=cuda)
            x = torch.randn(len(slots), T, D, generator=g).half().to(cuda)
            outs = []
            for st in states:
                batch = copy.copy(st)
                batch.cache = st.cache.batch(slots)
                batch.processed_frames, batch.cache_lengths = st.processed_frames[at], st.cache_lengths[at]
                out, batch = enc(x, batch, length=torch.full((len(slots),), T, dtype=torch.int64, device=cuda))
                st.processed_frames[at], st.cache_lengths[at] = batch.processed_frames, batch.cache_lengths
                outs.append(out)
            assert torch.equal(outs[0], outs[1])
    assert states[0].cache.pool.free_list().tolist() == states[1].cache.pool.free_list().tolist()


def _adapters(enc, G, r, seed, scale=0.7):
    """Random adapters of rank r and less, of every projection but one."""
    ad = EncoderAdapters(enc, G, 16)
    g = torch.Generator().manual_seed(seed)
    weights = []
    for i in range(G):
        w = {}
        for l in range(LY):
            for t in TARGETS[: 6 - i % 2]:
                n, k = enc.layers[l].get_submodule(t).weight.shape
                q = r - i
                w[f"layers.{l}.{t}"] = (torch.randn(q, k, generator=g) / math.sqrt(k), torch.randn(n, q, generator=g) / math.sqrt(q))
        ad.load(i, w, scale)
        weights.append(w)
    return ad, weights


def test_adapted_encoder_is_the_merged_encoders(cuda):
    """fp32: each stream's output is that of an encoder with its adapter merged into the
    weights.  Both sides are fp32: a product of K <= 256 terms is off by up to
    K 2^-24 of its absolute sum on either side, and the merged weight by its rounding;
    with some 20 products, norms and softmaxes one after another, each of whose branches
    has a gain of a few, 2^-24 * 256 * 2 * 20 * 8 = 5e-3 bounds outputs of order 1."""
    enc = _encoder(cuda, torch.float32)
    ad, weights = _adapters(enc, 3, 16, 11)
    merged = []
    for w in weights:
        m = copy.deepcopy(enc)
        for name, (a, b) in w.items():
            p = m.get_submodule(name).weight
            p.copy_((p.double().cpu() + 0.7 * b.double() @ a.double()).float())
        merged.append(m)
    merged.append(enc)
    ids = [2, -1, 0, 1, 2, 0]
    B = len(ids)
    new = lambda n: enc.init_streaming_state(batch_size=n, device=cuda, dtype=torch.float32, device_pages=True)  # noqa: E731
    state, alone = new(B), [new(1) for _ in ids]
    g = torch.Generator().manual_seed(8)
    dev_ids = torch.tensor(ids, dtype=torch.int32, device=cuda)
    apart = 0.0
    with torch.no_grad():
        for step in range(9):
            x = torch.randn(B, T, D, generator=g).to(cuda)
            one = torch.full((1,), T, dtype=torch.int64, device=cuda)
            got, state = enc(x, state, length=one.expand(B).contiguous(), adapters=ad.step(dev_ids, T))
            plain = None
            for b, i in enumerate(ids):
                want, alone[b] = merged[i](x[b : b + 1], alone[b], length=one)
                assert float((got[b] - want[0]).abs().max()) < 5e-3, (step, b)
                plain = want if plain is None else plain
            apart = max(apart, float((got[0] - got[1]).abs().max()))
    assert apart > 0.1


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_recorded_step_with_adapters(cuda, dtype):
    """Replays with the adapter numbers, and adapters loaded, changed between them: the
    eager step's bits."""
    enc = _encoder(cuda, dtype)
    ad, weights = _adapters(enc, 3, 8, 12)
    B = 6
    length = torch.full((B,), T, dtype=torch.int64, device=cuda)
    eager, replay = (enc.init_streaming_state(batch_size=B, device=cuda, dtype=dtype, device_pages=True) for _ in range(2))
    ids = torch.zeros(B, dtype=torch.int32, device=cuda)
    graph = EncoderStepGraph(enc, replay, length, adapters=ad, adapter_ids=ids)
    g = torch.Generator().manual_seed(9)
    outs = []
    with torch.no_grad():
        for step in range(8):
            x = torch.randn(B, T, D, generator=g).to(dtype).to(cuda)
            ids.copy_(torch.randint(-1, 4, (B,), generator=g).to(torch.int32))
            if step == 5:
                ad.load(1, weights[2], 0.3)
                ad.clear(0)
            want, _ = enc(x, eager, length=length, adapters=ad.step(ids, T))
            got = graph(x)
            assert torch.equal(got, want), step
            outs.append(got.clone())
            _same(eager, replay)
    assert torch.isfinite(torch.stack(outs)).all()


def test_adapter_bank_arguments(cuda):
    enc = _encoder(cuda, torch.float16)
    for bad in (dict(rank=12), dict(rank=136), dict(num_adapters=0), dict(num_adapters=513), dict(targets=("conv",))):
        with pytest.raises(ValueError):
            EncoderAdapters(enc, **(dict(num_adapters=2, rank=8) | bad))
    ad = EncoderAdapters(enc, 2, 8, targets=("self_attn.qkv",))
    a, b = torch.zeros(8, D), torch.zeros(3 * D, 8)
    with pytest.raises(IndexError):
        ad.load(2, {})
    with pytest.raises(KeyError):
        ad.load(0, {"layers.0.self_attn.linear_out": (a, b)})
    with pytest.raises(KeyError):
        ad.load(0, {"layers.7.self_attn.qkv": (a, b)})
    ad.load(0, {"layers.0.self_attn.qkv": (a + 1, b + 1)}, 2.0)
    with pytest.raises(ValueError):  # refused before anything changes
        ad.load(0, {"layers.0.self_attn.qkv": (torch.zeros(9, D), torch.zeros(3 * D, 9))})
    bank = ad.banks[0]["self_attn.qkv"]
    assert (bank.a[0] == 1).all() and bank.scale.tolist() == [2.0, 0.0]
    state = enc.init_streaming_state(batch_size=2, device=cuda, dtype=torch.float16)
    length = torch.full((2,), T, dtype=torch.int64, device=cuda)
    with pytest.raises(ValueError, match="go together"):
        EncoderStepGraph(enc, state, length, adapters=ad)
    with pytest.raises(ValueError, match="adapter_ids"):
        EncoderStepGraph(enc, state, length, adapters=ad, adapter_ids=torch.zeros(2, dtype=torch.int64, device=cuda))
    with pytest.raises(RuntimeError, match="device_pages"):
        state.cache.open_recorded_step()


def test_ragged_attention_step(cuda):
    """page_step -> adapter_linear (qkv) -> paged attention over the frames before the step
    and the stream's own new ones -> kv_append_slots, fp16, against the oracle on dense
    windows of the same q, k, v (bar 2e-3, the attention kernels' own)."""
    left, chunk, heads, dk, S = 23, 5, 2, 64, 8
    Dm, dt = heads * dk, torch.float16
    rng = np.random.default_rng(4)
    pool = DevicePagePool(S, 8, left, chunk, cuda)
    shape = synth.Shape("ragged", 1, Dm, heads, left=left, right=chunk - 1, page_size=8, dtype=dt)
    pos, bu, bv = synth.relpos_inputs(shape, cuda, seed=0)
    pages = lambda rows: ops.PagedKV(kp, vp, rows, pool.max_pages)  # noqa: E731
    kp, vp = (torch.full((1, pool.num_pages, 8, Dm), float("nan"), dtype=dt, device=cuda) for _ in range(2))
    g = torch.Generator(device=cuda).manual_seed(1)
    rnd = lambda *s, std=1.0: (torch.randn(s, generator=g, device=cuda) * std).to(dt)  # noqa: E731
    w = rnd(3 * Dm, Dm, std=Dm**-0.5)
    ad = ops.Adapters(rnd(4, 8, Dm, std=Dm**-0.5), rnd(4, 3 * Dm, 8, std=0.3), torch.full((4,), 1.5, device=cuda))
    said = [np.zeros((0, 2 * Dm)) for _ in range(S)]
    for step in range(16):
        slots = rng.permutation(S)[: rng.integers(1, S + 1)]
        B = len(slots)
        lengths = rng.integers(0, chunk + 1, B)
        ids = torch.from_numpy((slots % 5 - 1).astype(np.int32)).to(cuda)
        rows, place = pool.advance(slots, torch.from_numpy(lengths.astype(np.int32)).to(cuda))
        x = rnd(B, chunk, Dm)
        qkv = ops.adapter_linear(x, w, None, ad, ops.adapter_plan(ids, chunk, num_adapters=4))
        q, k, v = qkv.chunk(3, dim=-1)
        # masked: padding keys and queries, and positions before the stream's first frame
        A = np.array([len(said[s]) for s in slots])
        j = np.arange(left + chunk)[None, None, :]
        t = np.arange(chunk)[None, :, None]
        mask = (j < left - A[:, None, None]) | (j >= left + lengths[:, None, None]) | (t >= lengths[:, None, None])
        out = ops.paged_relpos_attn(q, k, v, pos, bu, bv, torch.from_numpy(mask).to(cuda), num_heads=heads, left=left, pages=pages(rows), append=False)
        ops.kv_append_slots(pages(rows), 0, k, v, place)
        kv = torch.cat([k, v], -1).double().cpu().numpy()
        win = np.zeros((B, left + chunk, 2 * Dm))
        for b, s in enumerate(slots):
            had = said[s][-left:]
            win[b, left - len(had) : left] = had
            win[b, left:] = kv[b]
            said[s] = np.concatenate([said[s], kv[b, : lengths[b]]])
        d = lambda a: a.double().cpu().numpy()  # noqa: E731
        want = oa.relpos_attention(d(q), win[..., :Dm], win[..., Dm:], d(pos), d(bu), d(bv), mask, heads)
        err = np.abs(d(out) - want)[np.arange(chunk)[None, :] < lengths[:, None]]
        assert err.size == 0 or err.max() < 2e-3, step
