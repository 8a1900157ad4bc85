"""Decode steps of the model over quantised caches and behind shared prefixes
(SyntheticDecoder.forward, KVCache.quantized / share) against the oracle's decode
steps, with the bars of the decode steps' own tests: per row cosine >= 0.9999 and max
error <= 1e-2 of the logits' scale, on the device's routing.

The oracle holds the cache's values (the codes times their scales) and quantises
each new token as the device does; a prefix is laid before the row's own
positions.  A K value next to a rounding border may get the neighbouring code on the
device (its float32 norm against the oracle's): one code of one token among many, far
inside the bars."""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

from oracle import decoder as od
from oracle import quant_cache as oq
from test_gpu_decoder import _check_logits, _to_np
from maple_amd.decode_graph import (BucketedDecodeGraphs, Sampling, _choose, batched_sampler_workspace, capture_decode_graph,
                                    generate, tree_step, try_decode_graph)
from maple_amd.model import DecoderConfig, SyntheticDecoder

pytestmark = pytest.mark.gpu

SMALL = DecoderConfig(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64, experts=8, inter=256,
                      top_k=2, vocab=1024, rtn_group=128, lm_scale=(0.01, 0.02))
MIXED = dataclasses.replace(SMALL, layer_types=("sliding_attention", "full_attention"), sliding_window=16,
                            nope_on_global=True)


def _values(kv):
    if len(kv) == 2:
        return kv[0].double().cpu().numpy(), kv[1].double().cpu().numpy()
    e = [t.view(torch.uint8).cpu().numpy().astype(np.int64) - 127 for t in kv[2:]]
    return tuple(oq.decode(c.double().cpu().numpy(), x) for c, x in zip(kv[:2], e))


def _joined(cache, rows):
    """The oracle's cache: each slot's prefix and own positions one after the other, in rows with room for both."""
    n = cache.seqlen.cpu().numpy()
    pos = cache.positions(len(rows)).cpu().numpy()
    more = 0 if cache.prefix is None else cache.prefix.max_len
    ks, vs = [], []
    for i in range(len(cache.k)):
        k, v = _values(cache.layer(i))
        shape = (len(rows), k.shape[1], k.shape[2] + more, k.shape[3])
        jk, jv = np.zeros(shape), np.zeros(shape)
        if cache.prefix is not None:
            pk, pv = _values(cache.prefix.layer(i, len(rows)).cache)
        for b, r in enumerate(rows):
            lead = pos[b] - n[b]
            if lead:
                p = int(cache.prefix.of[b])
                jk[b, :, :lead], jv[b, :, :lead] = pk[p, :, :lead], pv[p, :, :lead]
            jk[b, :, lead:lead + n[b]], jv[b, :, lead:lead + n[b]] = k[r, :, :n[b]], v[r, :, :n[b]]
        ks.append(jk)
        vs.append(jv)
    return dict(k=ks, v=vs, seqlen=pos.copy())


class _Quantising:
    """An oracle cache row that holds what it is given as the codes stand for it."""

    def __init__(self, rows):
        self.rows, self.shape = rows, rows.shape

    def __getitem__(self, at):
        got = self.rows[at]
        return _Quantising(got) if got.ndim == 3 else got

    def __setitem__(self, at, new):
        self.rows[at] = oq.decode(*oq.encode(np.asarray(new)))


def _steps(model, cache, ids, rows, n=3):
    """The device's steps against the oracle's, each from the device's cache and routing."""
    m = _to_np(model)
    for step in range(n):
        c = _joined(cache, rows)
        if cache.is_quantized:
            c["k"], c["v"] = [_Quantising(k) for k in c["k"]], [_Quantising(v) for v in c["v"]]
        routing = []
        logits = model.forward(ids, cache, routing)
        ref, _ = od.decoder_step(m, c, ids.cpu().numpy(), router_ids=[r.cpu().numpy() for r in routing])
        _check_logits(logits, ref, f"step {step}")
        ids = torch.argmax(logits, dim=-1)


def _ids(dev, batch, seed=3):
    return torch.randint(0, SMALL.vocab, (batch,), device=dev, generator=torch.Generator(device=dev).manual_seed(seed))


@pytest.mark.parametrize("cfg", [SMALL, MIXED], ids=["full", "sliding and NoPE"])
@pytest.mark.parametrize("batch", [1, 3, 20])
def test_steps_over_a_quantised_cache(dev, cfg, batch):
    model = SyntheticDecoder(cfg, dev, seed=5, max_len=128)
    cache = model.make_cache(batch, prefill_len=37, seed=1, quantized=True)
    _steps(model, cache, _ids(dev, batch), list(range(batch)))
    assert cache.seqlen.tolist() == [40] * batch


@pytest.mark.parametrize("cfg", [SMALL, MIXED], ids=["full", "sliding and NoPE"])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("batch", [1, 5])
def test_steps_behind_prefixes(dev, cfg, quantized, batch):
    model = SyntheticDecoder(cfg, dev, seed=6, max_len=256)
    cache = model.make_cache(batch + 1, prefill_len=90, seed=2, quantized=quantized, max_len=120)
    cache.share([batch, 0], [77, 31])
    cache.remap = True
    for slot in range(batch):
        cache.prefix.of[slot] = (0, 1, -1, 0, 0)[slot]
        cache.seqlen[slot] = (0, 7, 55, 33, 1)[slot]
    _steps(model, cache, _ids(dev, batch), list(range(batch)))


@pytest.mark.parametrize("quantized,longest", [(False, 2048), (True, 4096)])
def test_steps_behind_a_long_prefix(dev, quantized, longest):
    """At these sizes a prefix is read once for all of its rows."""
    batch = 32
    model = SyntheticDecoder(SMALL, dev, seed=8, max_len=longest + 64)
    source = model.make_cache(1, prefill_len=longest, seed=4, quantized=quantized, max_len=longest)
    cache = model.make_cache(batch, prefill_len=20, seed=5, quantized=quantized, max_len=64)
    cache.prefix = source.share([0], [longest - 3])
    cache.prefix.of = torch.zeros(batch, device=dev, dtype=torch.int64)
    cache.prefix.of[5] = -1
    cache.seqlen.copy_(torch.arange(batch, device=dev) % 21)
    _steps(model, cache, _ids(dev, batch), list(range(batch)), n=2)


def test_steps_through_a_slot_map(dev):
    model = SyntheticDecoder(SMALL, dev, seed=7, max_len=256)
    cache = model.make_cache(4, prefill_len=50, seed=3, quantized=True, max_len=100)
    cache.share([3], [50])
    cache.remap = True
    cache.prefix.of.copy_(torch.tensor([-1, 0, 0, -1], device=dev))
    cache.seqlen.copy_(torch.tensor([50, 3, 0, 10], device=dev))
    cache.swap_slots(0, 2)
    assert cache.prefix.of.tolist() == [0, 0, -1, -1] and cache.seqlen.tolist() == [0, 3, 50, 10]
    _steps(model, cache, _ids(dev, 3), [2, 1, 0])
    cache.reset_slot(1)
    assert cache.prefix.of[1] == -1 and cache.seqlen[1] == 0


def test_quantised_values_are_the_caches(dev):
    model = SyntheticDecoder(SMALL, dev, seed=5, max_len=64)
    a = model.make_cache(3, prefill_len=20, seed=1)
    b = a.quantized()
    back = b.dequantized()
    for i in range(SMALL.layers):
        ref = [oq.decode(*oq.encode(t.double().cpu().numpy())) for t in (a.k[i], a.v[i])]
        for got, want in zip((back.k[i], back.v[i]), ref):
            assert (got.double().cpu().numpy() == want).all()
    assert b.seqlen.tolist() == a.seqlen.tolist() and b.seqlen is not a.seqlen
    logits = model.forward(_ids(dev, 3), back)  # an ordinary cache
    assert torch.isfinite(logits.float()).all()


@pytest.mark.parametrize("quantized,prefix", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("sampling", [Sampling(), Sampling(temperature=0.8, top_p=0.9, top_k=20)], ids=["greedy", "drawn"])
def test_captured_steps_equal_eager_ones(dev, quantized, prefix, sampling):
    model = SyntheticDecoder(SMALL, dev, seed=9, max_len=256)
    if not sampling.greedy:
        sampling = dataclasses.replace(sampling, generator=torch.Generator(device=dev).manual_seed(5))

    def cache():
        c = model.make_cache(3, prefill_len=30, seed=2, quantized=quantized, max_len=100)
        if prefix:
            c.share([2], [30])
            c.prefix.of[:2] = 0
        return c

    logs = []
    c = cache()
    before = {k: ([t.clone() for t in v] if isinstance(v, list) else v) for k, v in c.snapshot().items()}
    g = try_decode_graph(model, c, _ids(dev, 3), sampling, log=logs.append)
    assert g is not None, logs
    after = c.snapshot()
    for n in ("k", "v") + (("k_scale", "v_scale") if quantized else ()):  # the cache is as it was
        assert all(torch.equal(x, y) for x, y in zip(before[n], after[n]))
    graph = generate(model, c, _ids(dev, 3), 6, Sampling())
    assert len(graph.token_ids) == 3 and all(len(t) == 6 for t in graph.token_ids)


@pytest.mark.parametrize("quantized,prefix", [(True, 0), (False, 30), (True, 30), (False, 2045), (True, 4093)],
                         ids=["quantised", "bf16, prefix", "quantised, prefix", "bf16, long prefix", "quantised, long prefix"])
@pytest.mark.parametrize("sampling", [Sampling(), Sampling(temperature=0.8, top_p=0.9, top_k=20)], ids=["greedy", "drawn"])
def test_captured_steps_repeat_eager_ones_to_the_bit(dev, quantized, prefix, sampling):
    """Logits, ids, write positions and every byte of the cache after each of six steps, replayed with eager work between
    them, against the same steps run eagerly; the long prefixes are read once for all of their rows."""
    rows = 32 if prefix > 1000 else 3
    model = SyntheticDecoder(SMALL, dev, seed=9, max_len=max(256, prefix + 64))
    cache = model.make_cache(rows, prefill_len=30, seed=2, quantized=quantized, max_len=64)
    if prefix:
        source = model.make_cache(1, prefill_len=prefix, seed=3, quantized=quantized, max_len=prefix)
        cache.prefix = source.share([0], [prefix])
        cache.prefix.of = torch.zeros(rows, device=dev, dtype=torch.int64)
        cache.prefix.of[1] = -1
        cache.seqlen.copy_(torch.arange(rows, device=dev) % 31)
    if not sampling.greedy:
        sampling = dataclasses.replace(sampling, generator=torch.Generator(device=dev))
    first, snap, n = _ids(dev, rows), cache.snapshot(), 6

    def state():
        raw = [t.view(torch.uint8 if t.element_size() == 1 else torch.int16) for i in range(SMALL.layers) for t in cache.layer(i)]
        return [cache.seqlen.clone()] + [t.clone() for t in raw]

    def start():
        cache.restore(snap)
        if sampling.generator is not None:
            sampling.generator.manual_seed(5)

    start()
    before, eager, tok, out = state(), [], first.clone(), torch.empty_like(first)
    ws = None if sampling.greedy else batched_sampler_workspace(SMALL.vocab, sampling.top_k, rows, dev)[0]
    for _ in range(n):
        u = None if sampling.greedy else sampling.draw(rows, dev)
        logits = model.forward(tok, cache)
        _choose(logits, sampling, out, u, ws)
        tok.copy_(out)
        eager.append([logits.clone(), out.clone()] + state())
    start()
    assert all(torch.equal(a, b) for a, b in zip(before, state()))
    g = capture_decode_graph(model, cache, first.clone(), sampling)
    start()
    g.token_ids.copy_(first)
    for step in range(n):
        ids = g.step(sampling)
        other = torch.randn(1 << 16, device=dev).sum()  # eager work on the same allocator
        torch.cuda.synchronize()
        got = [g.logits, ids] + state()
        assert all(torch.equal(a, b) for a, b in zip(eager[step], got)), step
        assert torch.isfinite(other)
    # each step wrote each row's token into every layer, and nothing else
    at, was, now = before[0], before[1:], state()[1:]
    for a, b in zip(was, now):
        new = (torch.arange(64, device=dev) >= at.view(-1, 1)) & (torch.arange(64, device=dev) < at.view(-1, 1) + n)
        mask = new.unsqueeze(1).expand(-1, SMALL.kv_heads, -1)
        assert torch.equal(a[~mask], b[~mask])
        if a.ndim == 4:
            assert (a[mask] != b[mask]).any(-1).all()


def test_bucketed_graphs_over_a_quantised_cache(dev):
    model = SyntheticDecoder(SMALL, dev, seed=9, max_len=256)
    c = model.make_cache(4, prefill_len=30, seed=2, quantized=True, max_len=100)
    c.share([3], [25])
    c.remap = True
    graphs = BucketedDecodeGraphs(model, c, widths=(2, 4), sampling=Sampling())
    c.prefix.of.copy_(torch.tensor([0, -1, 0, -1], device=dev))
    ids = _ids(dev, 4)
    for live in (2, 4, 1, 3):
        snap = c.snapshot()
        got = graphs.replay_logits(ids[:live]).clone()
        c.restore(snap)
        # (a narrower batch runs other kernels elsewhere in the model: the same width)
        w = graphs.width_for(live)
        want = model.forward(torch.cat([ids[:live], ids.new_zeros(w - live)]), c)[:live]
        assert torch.equal(got, want)


def test_trees_and_short_tables_are_refused(dev):
    model = SyntheticDecoder(SMALL, dev, seed=9, max_len=64)
    c = model.make_cache(2, prefill_len=30, seed=2, quantized=True)
    tokens, parents = torch.zeros(2, 3, device=dev, dtype=torch.int64), torch.tensor([[-1, 0, 1]] * 2, device=dev)
    for call in (lambda: model.forward_tree(tokens, parents, c), lambda: tree_step(model, c, tokens, parents)):
        with pytest.raises(ValueError, match="drafted trees"):
            call()
    p = model.make_cache(2, prefill_len=30, seed=2)
    p.share([0], [30])
    with pytest.raises(ValueError, match="drafted trees"):
        p.commit(tokens.int(), tokens[:, 0].int())
    with pytest.raises(ValueError, match="max_len"):
        model.forward(_ids(dev, 2), p)
    for bad in (lambda: p.share([0], [3]), lambda: c.quantized(), lambda: p.quantized(), lambda: p.dequantized(),
                lambda: c.share([2], [3]), lambda: c.share([0], [0]), lambda: c.share([], []), lambda: c.share([0], [1, 2])):
        with pytest.raises(ValueError):
            bad()
