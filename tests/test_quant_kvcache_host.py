"""The host's part of quantised KV caches and shared prefixes (KVCache), on the CPU."""

from __future__ import annotations

import weakref

import pytest
import torch

from maple_amd import model as model_module
from maple_amd import synthetic
from maple_amd.kernels import KV, QuantKV, make_quant_kv
from maple_amd.model import DecoderConfig, KVCache, SyntheticDecoder

LAYERS, ROWS, NKV, N, D = 2, 4, 2, 16, 64


def _plain():
    g = torch.Generator().manual_seed(1)
    ks, vs = ([torch.randn(ROWS, NKV, N, D, generator=g).bfloat16() for _ in range(LAYERS)] for _ in range(2))
    return KVCache(ks, vs, torch.tensor([3, 9, 0, 16]), N)


def _quant():
    g = torch.Generator().manual_seed(2)
    layers = [make_quant_kv(ROWS, NKV, N, D, "cpu") for _ in range(LAYERS)]
    for t in (t for c in layers for t in c):
        b = t.view(torch.uint8)
        b.copy_(torch.randint(1, 120, b.shape, generator=g))
    k, v, ks, vs = ([c[i] for c in layers] for i in range(4))
    return KVCache(k, v, torch.tensor([3, 9, 0, 16]), N, k_scale=ks, v_scale=vs)


MAKE = pytest.mark.parametrize("make", [_plain, _quant], ids=["bf16", "quantised"])


def _raw(t):
    return t.view(torch.uint8 if t.element_size() == 1 else torch.int16)


@MAKE
def test_layers_are_of_the_caches_kind(make):
    c = make()
    kv = c.layer(1)
    assert type(kv) is (QuantKV if c.is_quantized else KV)
    assert kv.k is c.k[1] and kv.v is c.v[1]
    if c.is_quantized:
        assert kv.k_scale is c.k_scale[1] and kv.v_scale is c.v_scale[1]


@MAKE
def test_share_copies_the_rows(make):
    c = make()
    want = [[_raw(t)[[3, 1], :, :9].clone() for t in c.layer(i)] for i in range(LAYERS)]
    p = c.share([3, 1], [9, 4])
    for t in (t for i in range(LAYERS) for t in c.layer(i)):
        _raw(t).zero_()  # the rows are free again
    assert p is c.prefix and p.max_len == 9 and p.length.tolist() == [9, 4] and p.of.tolist() == [-1] * ROWS
    for i in range(LAYERS):
        kv = p.layer(i, 3)
        assert type(kv.cache) is type(c.layer(i)) and kv.of.tolist() == [-1] * 3
        for got, ref in zip(kv.cache, want[i]):
            assert got.is_contiguous() and torch.equal(_raw(got), ref)


@MAKE
def test_positions_count_the_prefix(make):
    c = make()
    assert c.positions(3).tolist() == [3, 9, 0]
    c.share([3, 1], [9, 4])
    assert c.positions(4).tolist() == [3, 9, 0, 16]
    c.prefix.of.copy_(torch.tensor([0, 1, -1, 2]))  # (2: no prefix's index)
    assert c.positions(4).tolist() == [12, 13, 0, 16] and c.positions(2).tolist() == [12, 13]


@pytest.mark.parametrize("rows,lengths", [([], []), ([0, 1], [3]), ([4], [3]), ([-1], [3]), ([0], [0]), ([0], [17])])
def test_share_refuses(rows, lengths):
    with pytest.raises(ValueError, match="share"):
        _plain().share(rows, lengths)


def test_share_only_once():
    c = _plain()
    c.share([0], [3])
    with pytest.raises(ValueError, match="already"):
        c.share([1], [3])


@MAKE
def test_slots_carry_their_prefix(make):
    c = make()
    c.share([3, 1], [9, 4])
    c.prefix.of.copy_(torch.tensor([0, 1, -1, 0]))
    c.remap = True
    c.swap_slots(0, 2)
    assert c.prefix.of.tolist() == [-1, 1, 0, 0] and c.seqlen.tolist() == [0, 9, 3, 16]
    assert c.row_map.tolist() == [2, 1, 0, 3]
    c.reset_slot(1)
    assert c.prefix.of.tolist() == [-1, -1, 0, 0] and c.seqlen.tolist() == [0, 0, 3, 16]


@MAKE
@pytest.mark.parametrize("steps", [None, 4])
def test_snapshots_hold_scales_and_prefixes(make, steps):
    c = make()
    c.share([3], [9])
    c.prefix.of[1] = 0
    snap = c.snapshot(steps)
    lo, hi = snap["span"]
    before = [[_raw(t).clone() for t in c.layer(i)] for i in range(LAYERS)]
    for i in range(LAYERS):
        for t in c.layer(i):
            _raw(t)[:, :, lo:hi] = 7
    c.seqlen.add_(1)
    c.prefix.of.fill_(0)
    c.restore(snap)
    assert c.seqlen.tolist() == [3, 9, 0, 16] and c.prefix.of.tolist() == [-1, 0, -1, -1]
    for i in range(LAYERS):
        for t, ref in zip(c.layer(i), before[i]):
            assert torch.equal(_raw(t), ref)


def test_a_snapshot_without_prefixes_takes_none_back():
    c = _plain()
    snap = c.snapshot()
    c.share([3], [9])
    c.prefix.of.fill_(0)
    c.restore(snap)
    assert c.prefix.of.tolist() == [-1] * ROWS


def test_what_has_no_form_is_refused():
    c, q = _plain(), _quant()
    with pytest.raises(ValueError, match="bf16 cache"):
        q.quantized()
    with pytest.raises(ValueError, match="quantised cache"):
        c.dequantized()
    path, accepted = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="drafted trees"):
        q.commit(path, accepted)
    c.share([0], [3])
    q.share([0], [3])
    for make in (c.quantized, q.dequantized):
        with pytest.raises(ValueError, match="without shared prefixes"):
            make()
    with pytest.raises(ValueError, match="drafted trees"):
        c.commit(path, accepted)


def _decoder(max_len=N):
    """A decoder without weights: what ``make_cache`` reads of it."""
    m = SyntheticDecoder.__new__(SyntheticDecoder)
    m.cfg = DecoderConfig(layers=5, heads=4, kv_heads=NKV, head_dim=D)
    m.device, m.max_len = torch.device("cpu"), max_len
    return m


def test_a_quantised_cache_is_made_layer_by_layer(monkeypatch):
    """No layer's bf16 K and V outlive their quantisation: a cache that only fits quantised can be made."""
    made, seen, randn = [], [], synthetic.randn_bf16

    def make(*args):
        t = randn(*args)
        made.append(weakref.ref(t))
        return t

    def quantize(k, v, cache):
        live = [t for t in (r() for r in made) if t is not None]
        assert len(live) == 2 and live[0] is k and live[1] is v
        assert k.shape == v.shape == (ROWS, NKV, N, D) and not k[:, :, 9:].any() and k[:, :, :9].any()
        seen.append((_raw(k).clone(), _raw(v).clone(), cache))
        return cache

    monkeypatch.setattr(synthetic, "randn_bf16", make)
    monkeypatch.setattr(model_module, "quantize_kv", quantize)
    c = _decoder().make_cache(ROWS, 9, seed=3, quantized=True)
    assert len(made) == 10 and all(r() is None for r in made)
    assert c.is_quantized and c.max_len == N and c.seqlen.tolist() == [9] * ROWS and len(seen) == 5
    plain = _decoder().make_cache(ROWS, 9, seed=3)  # the same values
    for i, (k, v, kv) in enumerate(seen):
        assert all(a is b for a, b in zip(c.layer(i), kv))
        assert torch.equal(k, _raw(plain.k[i])) and torch.equal(v, _raw(plain.v[i]))


def test_quantised_caches_hold_no_workspace_of_bf16_steps(monkeypatch):
    monkeypatch.setattr(model_module, "quantize_kv", lambda k, v, cache: cache)
    c = _plain()
    c.attn_ws = torch.zeros(8)
    assert c.quantized().attn_ws is None
    assert _decoder().make_cache(ROWS, 9, quantized=True).attn_ws is None
    assert _decoder().make_cache(ROWS, 9).attn_ws is not None
