"""Steps over drafted trees through the model (SyntheticDecoder.forward_tree,
decode_graph.tree_step, KVCache.commit) against the oracle's decode steps along
each branch, with the bars of the decode steps' own tests: per row cosine >=
0.9999 and max error <= 1e-2 of the logits' scale, on the device's routing (the
choice of experts jumps where two are tied up to rounding)."""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

from oracle import decoder as od
from oracle import tree as ot
from test_gpu_decoder import _cache_np, _check_logits, _step_with_device_routing, _to_np
from maple_amd.decode_graph import Sampling, tree_step
from maple_amd.model import DecoderConfig, RopeScaling, SyntheticDecoder

pytestmark = pytest.mark.gpu

SMALL = DecoderConfig(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=64, experts=8, inter=256,
                      top_k=2, vocab=1024, rtn_group=128, lm_scale=(0.01, 0.02))
MIXED = dataclasses.replace(SMALL, layer_types=("sliding_attention", "full_attention"), sliding_window=16,
                            nope_on_global=True)
SCALED = dataclasses.replace(SMALL, rope_scaling=RopeScaling("yarn", 8.0, original_len=64))

#: rows of 9 nodes: a branching tree, a chain, a bush with padding, no sequence
TREES = np.array([[-1, 0, 0, 1, 1, 2, 3, 3, 6], [-1, 0, 1, 2, 3, 4, 5, 6, 7], [-1, 0, 0, 0, -1, 2, 4, -1, 5],
                  [-2, 0, 0, 0, 0, 0, 0, 0, 0]])


def _setup(dev, cfg, rows, prefill=37, seed=5):
    model = SyntheticDecoder(cfg, dev, seed=seed, max_len=128)
    return model, model.make_cache(rows, prefill_len=prefill, seed=1)


def _tokens(dev, w, t, seed=3):
    return torch.randint(0, SMALL.vocab, (w, t), device=dev, generator=torch.Generator(device=dev).manual_seed(seed))


def _oracle_logits(m, cache, rows, tokens, parents, routing):
    """Per node the oracle's logits after ordinary steps along its branch (None:
    padding); ``cache`` as it was before, ``rows[b]`` its row of K/V."""
    w, t = parents.shape
    lines = [ot.branches(p) for p in parents]
    nodes = [(b, i) for b in range(w) for i in range(t) if lines[b][i] is not None]
    c = dict(k=[k[[rows[b] for b, _ in nodes]] for k in cache["k"]],
             v=[v[[rows[b] for b, _ in nodes]] for v in cache["v"]],
             seqlen=np.array([cache["seqlen"][b] for b, _ in nodes]))
    out = [[None] * t for _ in range(w)]
    for s in range(max(len(lines[b][i]) for b, i in nodes)):
        # (a branch that has ended repeats its last node, unread)
        at = [(b, lines[b][i][min(s, len(lines[b][i]) - 1)]) for b, i in nodes]
        logits, _ = od.decoder_step(m, c, [tokens[b, j] for b, j in at],
                                    router_ids=[np.stack([r[b, j] for b, j in at]) for r in routing])
        for n, (b, i) in enumerate(nodes):
            if len(lines[b][i]) == s + 1:
                out[b][i] = logits[n]
    return out


@pytest.mark.parametrize("cfg", [SMALL, MIXED, SCALED], ids=["full", "sliding+nope", "scaled"])
@pytest.mark.parametrize("rows,remap", [(4, False), (6, True)])
def test_forward_tree_vs_oracle_branches(dev, cfg, rows, remap):
    model, cache = _setup(dev, cfg, rows)
    if remap:
        cache.remap = True
        cache.swap_slots(0, 5)
        cache.swap_slots(2, 4)
    w, t = TREES.shape
    cache.seqlen[:w] -= torch.tensor([0, 17, 36, 2], device=dev)
    m, before = _to_np(model), _cache_np(cache)
    tokens, parents = _tokens(dev, w, t), torch.tensor(TREES, device=dev, dtype=torch.int32)
    routing = []
    logits = model.forward_tree(tokens, parents, cache, routing=routing)
    assert logits.shape == (w, t, cfg.vocab) and logits.dtype == torch.bfloat16
    assert np.array_equal(cache.seqlen.cpu().numpy(), before["seqlen"])
    rows_of = cache.row_map[:w].tolist()
    ref = _oracle_logits(m, before, rows_of, tokens.cpu().numpy(), TREES,
                         [r.reshape(w, t, -1).cpu().numpy() for r in routing])
    for b in range(w):
        for i in range(t):
            if ref[b][i] is not None:
                _check_logits(logits[b, i][None], ref[b][i][None], f"row {b} node {i}")
    # only the nodes' places were written
    for new, old in zip(cache.k + cache.v, before["k"] + before["v"]):
        keep = np.ones(new.shape, bool)
        for b in range(w):
            if TREES[b, 0] == -1:
                s = int(before["seqlen"][b])
                keep[rows_of[b], :, s:s + t] = False
        np.testing.assert_array_equal(new.float().cpu().numpy()[keep], old[keep])


@pytest.mark.parametrize("sampling", [Sampling(), Sampling(temperature=0.9, top_p=0.95, top_k=20)],
                         ids=["greedy", "sampled"])
def test_tree_step_keeps_the_accepted_branch(dev, sampling):
    """A step's tokens are the oracle's verdict on the device's logits, its cache
    the accepted branch moved together, and ordinary decoding goes on from there."""
    w, t = TREES.shape
    model, cache = _setup(dev, MIXED, w)
    m = _to_np(model)
    parents = torch.tensor(TREES, device=dev, dtype=torch.int32)
    tokens = _tokens(dev, w, t)
    # draft the model's own choices along the chain row and one branch, so that some are accepted
    for _ in range(t):
        probe = model.forward_tree(tokens, parents, cache).float().argmax(-1)
        for b, i in ((1, j) for j in range(1, t)):
            tokens[b, i] = probe[b, int(TREES[b, i])]
        tokens[0, 1], tokens[0, 4] = probe[0, 0], probe[0, 1]
    tokens[1, 7] = (tokens[1, 7] + 1) % SMALL.vocab
    uniform = torch.rand(w, t, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    logits = model.forward_tree(tokens, parents, cache)
    before, seqlen = [x.clone() for x in cache.k + cache.v], cache.seqlen.clone()
    out = tree_step(model, cache, tokens, parents, sampling, uniform=uniform)
    kw = dict(temperature=1.0, top_p=1.0, top_k=1) if sampling.greedy else dict(
        temperature=sampling.temperature, top_p=sampling.top_p, top_k=sampling.top_k)
    for b in range(w):
        emitted, path = ot.verify(logits[b].double().cpu().numpy(), tokens[b].cpu().numpy(), TREES[b],
                                  uniform[b].cpu().numpy(), **kw)
        n = len(emitted)
        assert out.tokens[b].tolist() == emitted + [-1] * (t - n)
        assert out.path[b].tolist() == path + [-1] * (t - n)
        assert int(out.accepted[b]) == n - 1
        assert int(cache.seqlen[b]) == int(seqlen[b]) + n
        for new, old in zip(cache.k + cache.v, before):
            for j, node in enumerate(path):
                assert torch.equal(new[b, :, int(seqlen[b]) + j], old[b, :, int(seqlen[b]) + node])
    if sampling.greedy:
        assert out.accepted[:2].tolist() == [2, 6]
    live = int((out.accepted >= 0).sum())  # the rows without a sequence are last
    ids = out.tokens[torch.arange(live, device=dev), out.accepted[:live].long()]
    _step_with_device_routing(model, m, ids, cache, "after the commit", MIXED.top_k)


@pytest.mark.parametrize("rows", [1, 2])
def test_tree_steps_without_a_draft(dev, rows):
    """Greedy steps over a one-node tree (no draft) are ordinary greedy decoding:
    each step's logits meet the oracle's, and the token is their argmax."""
    model, cache = _setup(dev, SMALL, rows)
    m = _to_np(model)
    tok = torch.tensor([[7], [900]], device=dev)[:rows]
    parents = torch.full((rows, 1), -1, device=dev, dtype=torch.int32)
    for step in range(3):
        cnp, routing = _cache_np(cache), []
        logits = model.forward_tree(tok, parents, cache, routing=routing)
        ref, _ = od.decoder_step(m, cnp, tok.cpu().numpy(), router_ids=[r.cpu().numpy() for r in routing])
        _check_logits(logits[:, 0], ref, f"step {step}")
        out = tree_step(model, cache, tok, parents)
        assert out.accepted.tolist() == [0] * rows
        assert torch.equal(out.tokens[:, 0], logits[:, 0].argmax(-1))
        tok = out.tokens.clone()
    assert cache.seqlen.tolist() == [40] * rows


@pytest.mark.parametrize("w,t,top_k", [(1, 8, 1), (3, 9, 20), (4, 64, 20)])
def test_captured_tree_step_replays_as_eager(dev, w, t, top_k):
    """One graph of the whole step, fed from its buffers: every replay equals the
    eager step on the same inputs, with eager work between the replays, and a
    second captured graph of the same step in turn."""
    model, cache = _setup(dev, SMALL, w, prefill=20)
    sampling = Sampling(temperature=0.8, top_k=top_k)
    rng = np.random.default_rng(t)

    def inputs(step):
        p = np.full((w, t), -1)
        for b in range(w):
            for i in range(1, t - (b % 2)):
                p[b, i] = rng.integers(max(0, i - 3), i)
        g = torch.Generator(device=dev).manual_seed(step)
        return (torch.randint(0, SMALL.vocab, (w, t), device=dev, generator=g),
                torch.tensor(p, device=dev, dtype=torch.int32), torch.rand(w, t, device=dev, generator=g))

    steps = [inputs(s) for s in range(4)]
    start = [x.clone() for x in (*cache.k, *cache.v)]

    def rewind():
        cache.seqlen.fill_(20)
        for x, y in zip((*cache.k, *cache.v), start):
            x.copy_(y)

    def run(args):
        tok, par, u = args
        return tree_step(model, cache, tok, par, sampling, uniform=u)

    eager = []
    for s in steps[:2]:  # (64 nodes: two steps fit the cache)
        out = run(s)
        eager.append(([x.clone() for x in out], [x.clone() for x in (cache.seqlen, *cache.k, *cache.v)]))
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        rewind()
        bufs = [x.clone() for x in steps[2]]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            run(bufs)
        side.synchronize()
        rewind()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(bufs)
        graphs.append((g, bufs, out))
    for again in range(2):
        for g, bufs, out in graphs:
            rewind()
            for s, (want, state) in zip(steps, eager):
                for x, y in zip(bufs, s):
                    x.copy_(y)
                g.replay()
                torch.cuda.synchronize()
                for x, y in zip(out, want):
                    assert torch.equal(x, y)
                for x, y in zip((cache.seqlen, *cache.k, *cache.v), state):
                    assert torch.equal(x, y)
                torch.zeros(1, device=dev).add_(1)


@pytest.mark.parametrize("sampling", [Sampling(), Sampling(temperature=0.9, top_p=0.95, top_k=20)],
                         ids=["greedy", "sampled"])
def test_tree_step_near_the_caches_end(dev, sampling):
    """Rows with room for some nodes, for one and for none: a node whose K/V could
    not be stored is never accepted, whatever its token; a full row takes no step;
    no write position passes the cache's end."""
    model, cache = _setup(dev, SMALL, 4)
    room = [3, 0, 1, 60]
    cache.seqlen.copy_(128 - torch.tensor(room, device=dev))
    # nodes 1 .. 5 are unlikely; node 6 is the root's best token, node 7 the best behind it, node 8 behind that
    tree = np.array([[-1, 0, 0, 1, 1, 2, 0, 6, 7]] * 4)
    parents = torch.tensor(tree, device=dev)
    w, t = tree.shape
    tokens = _tokens(dev, w, t)
    full = cache.seqlen.clone()
    cache.seqlen.fill_(60)  # (any place with room: the tokens only have to be drafted well)
    for _ in range(4):
        probe = model.forward_tree(tokens, parents.int(), cache).float()
        for i in (6, 7, 8):
            tokens[:, i] = probe[:, tree[0, i]].argmax(-1)
        tokens[:, 1:3] = probe[:, :1].argmin(-1)
    cache.seqlen.copy_(full)
    fitted = np.where(full.cpu().numpy()[:, None] + np.arange(t) < 128, tree, -2)
    for _ in range(4):  # the same where the rows are now
        probe = model.forward_tree(tokens, torch.tensor(fitted, device=dev, dtype=torch.int32), cache).float()
        for i in (6, 7, 8):
            tokens[3, i] = probe[3, tree[0, i]].argmax(-1)
        tokens[:3, 6] = probe[:3, 0].argmax(-1)
        tokens[:, 1:3] = probe[:, :1].argmin(-1)
    logits = model.forward_tree(tokens, torch.tensor(fitted, device=dev, dtype=torch.int32), cache)
    before, seqlen = [x.clone() for x in cache.k + cache.v], cache.seqlen.tolist()
    uniform = torch.zeros(w, t, device=dev)  # (every token that is possible is accepted)
    out = tree_step(model, cache, tokens, parents, sampling, uniform=uniform)
    kw = dict(temperature=1.0, top_p=1.0, top_k=1) if sampling.greedy else dict(
        temperature=sampling.temperature, top_p=sampling.top_p, top_k=sampling.top_k)
    for b in range(w):
        emitted, path = ot.verify(logits[b].double().cpu().numpy(), tokens[b].cpu().numpy(), fitted[b],
                                  uniform[b].cpu().numpy(), **kw)
        n = len(emitted)
        assert out.tokens[b].tolist() == emitted + [-1] * (t - n), b
        assert out.path[b].tolist() == path + [-1] * (t - len(path)), b
        assert int(out.accepted[b]) == n - 1 and int(cache.seqlen[b]) == seqlen[b] + n <= 128, b
        for new, old in zip(cache.k + cache.v, before):
            assert torch.equal(new[b, :, :seqlen[b]], old[b, :, :seqlen[b]])
            for j, node in enumerate(path):
                assert torch.equal(new[b, :, seqlen[b] + j], old[b, :, seqlen[b] + node])
    assert out.accepted.tolist() == [0, -1, 0, 3]
    for _ in range(9):  # on to the end: the rows fill up and stay there
        out = tree_step(model, cache, tokens, parents, sampling, uniform=uniform)
        assert int(cache.seqlen.max()) <= 128
    assert cache.seqlen[:3].tolist() == [128] * 3 and out.accepted[:3].tolist() == [-1] * 3


def test_a_flash_head_scores_a_single_rows_tree(dev):
    """With a FlashHead, ordinary steps of one row are scored by it and steps of
    several rows by the exact head: so are trees, whatever their number of nodes."""
    from test_gpu_flash_head import _flash

    model, cache = _setup(dev, dataclasses.replace(SMALL, rtn_group=64), 1)
    two = model.make_cache(2, prefill_len=37, seed=1)
    flash = _flash(dev, model.lm_head, 32, 4, seed=4, force=(5,))[0]
    calls = []

    def spy(hidden, out=None):
        calls.append(hidden.clone())
        return flash(hidden, out=out)

    def trees(w, t):
        return _tokens(dev, w, t), torch.tensor(TREES[:w, :t], device=dev, dtype=torch.int32)

    for t in (1, 2, 9):
        tokens, parents = trees(1, t)
        model.flash_head = None
        exact = model.forward_tree(tokens, parents, cache)
        model.flash_head = spy
        calls.clear()
        logits = model.forward_tree(tokens, parents, cache)
        assert logits.shape == (1, t, SMALL.vocab) and len(calls) == t
        kept = logits.clone()
        for i, hidden in enumerate(calls):
            assert torch.equal(flash(hidden).reshape(-1), kept[0, i])
        assert torch.equal(logits, kept)  # (not the FlashHead's own row, which the next call overwrites)
        on = torch.isfinite(kept.float())
        assert (on.sum(-1) >= 4 * 32).all() and (on.sum(-1) <= 4 * 32 + 1).all() and on[..., 5].all()
        assert torch.isneginf(kept[~on].float()).all()
        got, ref = kept.float()[on], exact.float()[on]
        assert (got - ref).abs().max() <= 1e-2 * ref.abs().max()
        tokens, parents = trees(2, t)
        model.flash_head = None
        exact = model.forward_tree(tokens, parents, two)
        model.flash_head = spy
        calls.clear()
        assert torch.equal(model.forward_tree(tokens, parents, two), exact) and not calls
    # a whole step: the verdict is the law's on those logits
    tokens, parents = trees(1, 9)
    for sampling in (Sampling(), Sampling(temperature=0.9, top_p=0.95, top_k=20)):
        cache.seqlen.fill_(37)
        probe = model.forward_tree(tokens, parents, cache)
        tokens[0, 1] = probe[0, 0].float().argmax()
        logits = model.forward_tree(tokens, parents, cache)
        uniform = torch.full((1, 9), 0.25, device=dev)
        out = tree_step(model, cache, tokens, parents, sampling, uniform=uniform)
        kw = dict(temperature=1.0, top_p=1.0, top_k=1) if sampling.greedy else dict(
            temperature=sampling.temperature, top_p=sampling.top_p, top_k=sampling.top_k)
        emitted, path = ot.verify(logits[0].double().cpu().numpy(), tokens[0].cpu().numpy(), TREES[0],
                                  uniform[0].cpu().numpy(), **kw)
        assert out.tokens[0].tolist() == emitted + [-1] * (9 - len(emitted))
        assert out.path[0].tolist() == path + [-1] * (9 - len(path))
        if sampling.greedy:
            assert int(out.accepted[0]) >= 1


def test_a_captured_tree_step_with_a_flash_head_replays_as_eager(dev):
    from test_gpu_flash_head import _flash

    model, cache = _setup(dev, dataclasses.replace(SMALL, rtn_group=64), 1)
    model.flash_head = _flash(dev, model.lm_head, 32, 4, seed=4)[0]
    bufs, parents = _tokens(dev, 1, 5), torch.tensor(TREES[:1, :5], device=dev, dtype=torch.int32)
    run = lambda: tree_step(model, cache, bufs, parents)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for seed in range(4):
        tokens = _tokens(dev, 1, 5, seed=10 + seed)
        cache.seqlen.fill_(37)
        bufs.copy_(tokens)
        want = [x.clone() for x in (*run(), cache.seqlen, *cache.k, *cache.v)]
        cache.seqlen.fill_(37)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((*out, cache.seqlen, *cache.k, *cache.v), want):
            assert torch.equal(a, b), seed


def test_a_flash_heads_rows_of_any_vocabulary(dev):
    """A vocabulary that is no multiple of 8: the nodes' rows start where the
    FlashHead can write them."""
    from test_gpu_flash_head import _flash

    cfg = dataclasses.replace(SMALL, vocab=1028, rtn_group=64)
    model, cache = _setup(dev, cfg, 1)
    model.flash_head = _flash(dev, model.lm_head, 257, 40, seed=2)[0]
    tokens, parents = _tokens(dev, 1, 3), torch.tensor([[-1, 0, 0]], device=dev, dtype=torch.int32)
    logits = model.forward_tree(tokens, parents, cache)
    assert logits.shape == (1, 3, 1028) and (torch.isfinite(logits.float()).sum(-1) == 160).all()
    out = tree_step(model, cache, tokens, parents)
    best = logits.float().argmax(-1)
    assert int(out.tokens[0, 0]) == int(best[0, 0])
