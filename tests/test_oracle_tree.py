"""The tree-decoding oracle (oracle/tree.py) against hand-made cases, the
one-token oracles and the law that the verification has to keep (CPU)."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import decoder as od
from oracle import sampler as osm
from oracle import tree as ot


def test_branches_by_hand():
    assert ot.branches([-1, 0, 0, 1, 3, 2]) == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 1, 3, 4], [0, 2, 5]]
    # padding: a parent that is missing, itself, later or below an absent node
    assert ot.branches([-1, -1, 0, 1, 4, 9]) == [[0], None, [0, 2], None, None, None]
    assert ot.branches([0, 0]) == [None, None] and ot.branches([-2]) == [None]


def test_rotate_turns_each_pair_by_its_angle():
    rng = np.random.default_rng(0)
    y, a = rng.normal(size=16), rng.normal(size=3)
    cos, sin = np.cos(np.concatenate([a, a])), np.sin(np.concatenate([a, a]))
    for inter in (False, True):
        out, _ = ot.rotate(y, cos, sin, 6, inter)
        for i in range(3):
            p, q = (2 * i, 2 * i + 1) if inter else (i, i + 3)
            z = (y[p] + 1j * y[q]) * np.exp(1j * a[i])
            np.testing.assert_allclose([out[p], out[q]], [z.real, z.imag], rtol=1e-12, atol=1e-12)
        np.testing.assert_array_equal(out[6:], y[6:])


def test_one_node_is_the_one_token_step():
    rng = np.random.default_rng(1)
    cos, sin = od.rope_tables(32, 8, 10000.0)
    x, w = rng.normal(size=64), rng.uniform(0.5, 1.5, 64)
    got, _ = ot.head(x, w, cos[7], sin[7], 8, False, 1e-6)
    from oracle.kernels import bf16_round
    want = od.head_norm_rope(x, w, bf16_round(cos[7]), bf16_round(sin[7]), 8, 1e-6)
    np.testing.assert_allclose(got, want, rtol=1e-12)
    q, k, v = rng.normal(size=(4, 16)), rng.normal(size=(2, 20, 16)), rng.normal(size=(2, 20, 16))
    for window in (None, 5):
        got, _ = ot.attention(q, k, v, ot.seen([-1], 12, 20, window)[0], 0.25)
        np.testing.assert_allclose(got, od.gqa(q, k, v, 13, 0.25, window), rtol=2e-2, atol=2e-2)  # (its P is bf16)
    logits = rng.normal(size=50).astype(np.float32) * 2
    for u in (0.0, 0.3, 0.9):
        out, path = ot.verify([logits], [0], [-1], [u], temperature=0.8, top_p=0.9, top_k=20)
        assert path == [0] and out == [osm.sample_row(logits, u, temperature=0.8, top_p=0.9, top_k=20)]


def test_a_chain_attends_causally_and_windows_count_depth():
    assert ot.seen([-1, 0, 1, 2], 3, 100) == [[0, 1, 2, 3], [0, 1, 2, 3, 4], [0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 4, 5, 6]]
    # nodes 1 and 2 are siblings at position 4; node 3 below 2 at position 5
    assert ot.seen([-1, 0, 0, 2], 3, 100, 3) == [[1, 2, 3], [2, 3, 4], [2, 3, 5], [3, 5, 6]]
    assert ot.seen([-1, 0, -1], 3, 4, 1) == [[3], [], None]  # node 1's slot is past the cache's end


def _first_token_law(tree, probs, logits, choices, grid, **kw):
    """The law of the first emitted token: the draft's choices weighted by their
    probabilities, the uniforms over the midpoints of a grid."""
    v = logits.shape[1]
    law = np.zeros(v)
    u = (np.arange(grid) + 0.5) / grid
    for tokens, weight in choices:
        if len(tree) == 2:
            for a in u:
                for b in u:
                    law[ot.verify(logits, tokens, tree, [b, a], probs=probs, **kw)[0][0]] += weight / grid ** 2
        else:
            for a in u:
                for a2 in u:
                    for b in u:
                        law[ot.verify(logits, tokens, tree, [b, a, a2], probs=probs, **kw)[0][0]] += weight / grid ** 3
    return law


def test_verification_keeps_the_law():
    """One drawn child, two drawn siblings and a chosen child: the first token's
    law is the root's, to the grid's resolution (each of the draws is off by at
    most half a cell per token)."""
    rng = np.random.default_rng(2)
    v = 4
    logits = rng.normal(size=(3, v)) * 1.5
    q = rng.dirichlet(np.ones(v), size=2)
    kw = dict(temperature=0.9, top_p=1.0, top_k=4)
    ids, p = ot.law(logits[0], **kw)
    want = np.zeros(v)
    want[ids] = p
    one = [([0, t], q[0][t]) for t in range(v)]
    got = _first_token_law([-1, 0], np.stack([q[0], q[0]]), logits, one, 64, **kw)
    np.testing.assert_allclose(got, want, atol=2 * v / 64 / 2)
    two = [([0, s, t], q[0][s] * q[1][t]) for s in range(v) for t in range(v)]
    got = _first_token_law([-1, 0, 0], np.stack([q[0], q[0], q[1]]), logits, two, 16, **kw)
    np.testing.assert_allclose(got, want, atol=3 * v / 16 / 2)
    got = _first_token_law([-1, 0], None, logits, [([0, 2], 1.0)], 64, **kw)
    np.testing.assert_allclose(got, want, atol=2 * v / 64 / 2)


@pytest.mark.parametrize("drafted", [None, "uniform"])
def test_greedy_keeps_the_branch_of_argmaxes(drafted):
    rng = np.random.default_rng(3)
    logits = rng.normal(size=(5, 9))
    best = logits.argmax(1)
    tree = [-1, 0, 0, 2, 3]
    tokens = [0, (best[0] + 1) % 9, best[0], best[2], (best[3] + 1) % 9]
    probs = None if drafted is None else np.full((5, 9), 1.0 / 9)
    out, path = ot.verify(logits, tokens, tree, [0.5] * 5, temperature=1.0, top_p=1.0, top_k=1, probs=probs)
    assert path == [0, 2, 3] and out == [best[0], best[2], best[3]]


def test_the_law_of_infinite_logits():
    """+inf (a forced token) takes all of the mass, alike where there are several;
    rows of nothing but -inf weigh the first top_k tokens alike."""
    kw = dict(temperature=0.7, top_p=1.0, top_k=4)
    inf = np.inf
    ids, p = ot.law(np.array([1.0, inf, 3.0, -inf, 2.0]), **kw)
    assert ids.tolist() == [1, 2, 4, 0] and p.tolist() == [1.0, 0.0, 0.0, 0.0]
    ids, p = ot.law(np.array([inf, 1.0, inf, -inf, 2.0]), **kw)
    assert ids.tolist() == [0, 2, 4, 1] and p.tolist() == [0.5, 0.5, 0.0, 0.0]
    ids, p = ot.law(np.full(6, -inf), **kw)
    assert ids.tolist() == [0, 1, 2, 3] and p.tolist() == [0.25] * 4
    ids, p = ot.law(np.array([-inf, 0.0, -inf, 0.0, -inf]), **kw)
    assert ids.tolist() == [1, 3, 0, 2] and p.tolist() == [0.5, 0.5, 0.0, 0.0]
    for top_k in (1, 3):  # a drafted token that is forced is kept, whatever the uniform
        out, path = ot.verify(np.array([[0.0, 1.0, inf], [5.0, 1.0, 0.0]]), [0, 2], [-1, 0], [0.2, 0.999999],
                              temperature=1.0, top_p=0.9, top_k=top_k)
        assert path == [0, 1] and out == [2, 0]
