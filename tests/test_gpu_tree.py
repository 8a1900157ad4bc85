"""Decoding with trees of drafted tokens (kernels/tree.py) against the float64
oracle (oracle/tree.py).

Tolerances.  An output is rounded to bf16 once: 2^-8 of its value.  QKV: the
float32 norm and rotation are within 2^-16 of the sum of the terms' magnitudes
(a sum of at most 128 squares, a square root, a division and four products, each
within a few 2^-24).  Attention: each weight p is rounded to bf16 (2^-8 of it) in
the numerator and, alike, in the sum, so the quotient is off by at most 2 x 2^-8
of sum p |v| (the output is at most that too), and float32 scores, exponentials
and sums stay within another 2^-12 of it at these score sizes.  Verification and
commit are exact."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import tree as ot

pytestmark = pytest.mark.gpu

EPS = 1e-6


def np64(t):
    return t.detach().double().cpu().numpy()


def random_parents(rng, batch, nodes, ragged=True):
    p = np.full((batch, nodes), -1, np.int64)
    for b in range(batch):
        n = nodes if not ragged or b == 0 else int(rng.integers(1, nodes + 1))
        for i in range(1, n):
            p[b, i] = i - 1 if rng.random() < 0.4 else rng.integers(0, i)
    return p


def as_parents(p, dev):
    return torch.tensor(np.asarray(p), dtype=torch.int32, device=dev)


def bf16(dev, *shape, seed=0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16)


def tables(n, rot, dev, dtype=torch.float32):
    from maple_amd.model import rope_tables

    cos, sin = rope_tables(n, rot, 10000.0, dev)
    return cos.to(dtype), sin.to(dtype)


# ---------------------------------------------------------------------------
# QKV
# ---------------------------------------------------------------------------
def check_qkv(dev, parents, seqlen, heads, rot, *, interleaved=False, norm=True, max_len=64, rows=None, row_map=None,
              table=torch.float32, w_dtype=torch.float32, qkv=None, seed=0):
    from maple_amd.kernels import apply_qkv_tree

    nq, nkv, d = heads
    b, t = np.shape(parents)
    rows = rows or b
    if qkv is None:
        qkv = bf16(dev, b, t, (nq + 2 * nkv) * d, seed=seed)
    k, v = bf16(dev, rows, nkv, max_len, d, seed=seed + 1), bf16(dev, rows, nkv, max_len, d, seed=seed + 2)
    k0, v0 = k.clone(), v.clone()
    qw = kw = None
    if norm:
        qw = (torch.rand(d, device=dev) + 0.5).to(w_dtype)
        kw = (torch.rand(d, device=dev) + 0.5).to(w_dtype)
    cos, sin = tables(max_len + 64, max(rot, 2), dev, table)
    q = apply_qkv_tree(qkv, qw, kw, cos, sin, k, v, torch.tensor(seqlen, device=dev), as_parents(parents, dev),
                       row_map=None if row_map is None else torch.tensor(row_map, device=dev), num_heads=nq,
                       num_kv_heads=nkv, head_dim=d, rotary_dim=rot, use_rope=rot > 0, interleaved=interleaved, eps=EPS)
    assert q.shape == (b, t, nq, d) and q.dtype == torch.bfloat16
    qo, ko, vo, x = np64(q), np64(k), np64(v), np64(qkv).reshape(b, t, nq + 2 * nkv, d)
    k_left, v_left = np.ones(ko.shape[:1] + ko.shape[2:3], bool), np.ones(vo.shape[:1] + vo.shape[2:3], bool)
    c_np, s_np = np64(cos), np64(sin)
    for r in range(b):
        cr = r if row_map is None else row_map[r]
        for i, up in enumerate(ot.branches(parents[r])):
            if up is None:
                assert (qo[r, i] == 0).all()
                continue
            at = min(seqlen[r] + len(up) - 1, c_np.shape[0] - 1)
            slot = seqlen[r] + i
            for h in range(nq + nkv):
                if h >= nq and slot >= max_len:
                    continue
                w = None if not norm else np64(qw if h < nq else kw)
                ref, mag = ot.head(x[r, i, h], w, c_np[at], s_np[at], rot, interleaved, EPS)
                got = qo[r, i, h] if h < nq else ko[cr, h - nq, slot]
                assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -16 * mag + 1e-30).all(), (r, i, h)
            if slot < max_len:
                assert (vo[cr, :, slot] == x[r, i, nq + nkv:]).all()
                k_left[cr, slot] = v_left[cr, slot] = False
    for now, was, left in ((k, k0, k_left), (v, v0, v_left)):  # everything else is as it was, to the bit
        same = (now.view(torch.int16) == was.view(torch.int16)).all(dim=3).all(dim=1).cpu().numpy()
        assert same[left].all()
    return q


@pytest.mark.parametrize("heads", [(32, 4, 64), (16, 4, 128), (3, 1, 64), (2, 2, 128)])
@pytest.mark.parametrize("rot,interleaved", [(0, False), (2, True), (20, False), (20, True), (32, False), (32, True),
                                             (64, False), (64, True)])
def test_qkv_layouts_and_rotary_dims(dev, heads, rot, interleaved):
    rng = np.random.default_rng(rot)
    check_qkv(dev, random_parents(rng, 3, 7), [0, 5, 40], heads, rot, interleaved=interleaved)


@pytest.mark.parametrize("nodes", [1, 2, 33, 64])
def test_qkv_tree_sizes(dev, nodes):
    rng = np.random.default_rng(nodes)
    check_qkv(dev, random_parents(rng, 4, nodes), [0, 1, 3, 60], (8, 2, 128), 128, interleaved=True, max_len=128)


@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("w_dtype", [torch.float32, torch.bfloat16])
def test_qkv_table_and_weight_types(dev, table, w_dtype):
    check_qkv(dev, [[-1, 0, 0, 1]], [9], (4, 2, 64), 32, table=table, w_dtype=w_dtype)


def test_qkv_without_norm_strided_rows_and_row_map(dev):
    rng = np.random.default_rng(5)
    width = (4 + 2 * 2) * 64
    big = bf16(dev, 3, 9, width + 24, seed=9)
    for lo in (0, 3):  # aligned and unaligned rows
        check_qkv(dev, random_parents(rng, 3, 5), [0, 2, 7], (4, 2, 64), 32, norm=lo == 0,
                  qkv=big[:, 2:7, lo:lo + width], rows=6, row_map=[4, 0, 5])


def test_qkv_padding_rows_without_a_sequence_and_the_caches_end(dev):
    parents = [[-1, 0, -1, 2, 5, 0, -7, 1], [-2, 0, 1, 2, 3, 4, 5, 6], [-1, 0, 1, 2, 3, 4, 5, 6]]
    check_qkv(dev, parents, [3, 4, 59], (4, 2, 64), 64, max_len=64)  # the third row has room for 5 of its 8
    check_qkv(dev, parents, [3, 4, 64], (4, 2, 64), 64, max_len=64)  # and for none


def test_one_node_is_apply_qkv_decode(dev):
    """A tree of one node against the one-token call: the same arithmetic but for
    the order in which the squares are summed, so at most one bf16 step apart, and
    nearly always equal."""
    from maple_amd.kernels import apply_qkv_decode, apply_qkv_tree

    nq, nkv, d, rot = 32, 4, 64, 32
    b = 5
    qkv = bf16(dev, b, (nq + 2 * nkv) * d)
    qw, kw = torch.rand(d, device=dev) + 0.5, torch.rand(d, device=dev) + 0.5
    sl = torch.tensor([0, 1, 17, 100, 127], device=dev)
    cos, sin = tables(128, rot, dev)
    k1, v1 = bf16(dev, b, nkv, 128, d, seed=1), bf16(dev, b, nkv, 128, d, seed=2)
    k2, v2 = k1.clone(), v1.clone()
    kw_ = dict(num_heads=nq, num_kv_heads=nkv, head_dim=d, rotary_dim=rot, use_rope=True, eps=EPS)
    q1 = apply_qkv_decode(qkv, qw, kw, cos[sl], sin[sl], k1, v1, sl, use_qk_norm=True, **kw_)
    q2 = apply_qkv_tree(qkv.unsqueeze(1), qw, kw, cos, sin, k2, v2, sl, as_parents([[-1]] * b, dev), **kw_)
    assert torch.equal(v1, v2)
    for a, c in ((q1.reshape(-1), q2.reshape(-1)), (k1.reshape(-1), k2.reshape(-1))):
        off = (a.float() - c.float()).abs()
        assert (off <= 2.0 ** -7 * a.float().abs()).all() and (off > 0).float().mean() < 0.01


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def check_attention(dev, parents, seqlen, heads, *, window=None, max_len=None, rows=None, row_map=None, seed=0,
                    spoil=None, k=None, v=None, scale=None):
    """``spoil(k, v)``: values put into the caches that only the oracle's seen
    positions may carry on."""
    from maple_amd.kernels import tree_attention

    nq, nkv, d = heads
    b, t = np.shape(parents)
    max_len = max_len or max(seqlen) + t
    rows = rows or b
    q = bf16(dev, b, t, nq, d, seed=seed)
    if k is None:
        k, v = bf16(dev, rows, nkv, max_len, d, seed=seed + 1), bf16(dev, rows, nkv, max_len, d, seed=seed + 2)
    if spoil:
        spoil(k, v)
    scale = scale or d ** -0.5
    out = tree_attention(q, k, v, torch.tensor(seqlen, device=dev), as_parents(parents, dev), scale=scale,
                         row_map=None if row_map is None else torch.tensor(row_map, device=dev), window=window)
    assert out.shape == q.shape and out.dtype == torch.bfloat16
    compare_attention(out, q, k, v, parents, seqlen, scale, window, row_map)
    return out


def compare_attention(out, q, k, v, parents, seqlen, scale, window=None, row_map=None):
    got, qn = np64(out), np64(q)
    for r in range(q.shape[0]):
        cr = r if row_map is None else row_map[r]
        kn, vn = np64(k[cr]), np64(v[cr])
        for i, at in enumerate(ot.seen(parents[r], seqlen[r], k.shape[2], window)):
            if at is None:
                assert (got[r, i] == 0).all(), (r, i)
                continue
            with np.errstate(invalid="ignore"):
                ref, mag = ot.attention(qn[r, i], kn, vn, at, scale)
            fine = np.isfinite(ref)
            assert (np.isnan(got[r, i]) == np.isnan(ref)).all() and (got[r, i][~fine & ~np.isnan(ref)]
                                                                     == ref[~fine & ~np.isnan(ref)]).all(), (r, i)
            bound = (2.0 ** -8 * np.abs(ref) + (2.0 ** -7 + 2.0 ** -12) * mag)[fine]
            err = np.abs(got[r, i] - ref)[fine]
            assert (err <= bound + 1e-30).all(), (r, i, float((err - bound).max()))


@pytest.mark.parametrize("heads", [(32, 4, 64), (16, 4, 128), (4, 4, 64), (16, 1, 128), (5, 1, 64)])
@pytest.mark.parametrize("nodes", [1, 2, 5, 17, 64])
def test_attention_head_layouts_and_tree_sizes(dev, heads, nodes):
    rng = np.random.default_rng(nodes)
    check_attention(dev, random_parents(rng, 3, nodes), [0, 130, 257], heads)


@pytest.mark.parametrize("length", [0, 1, 31, 32, 33, 63, 64, 100, 127, 128, 129, 511, 1000, 2049])
@pytest.mark.parametrize("heads", [(8, 1, 64), (4, 2, 128)])
def test_attention_lengths(dev, length, heads):
    rng = np.random.default_rng(length)
    check_attention(dev, random_parents(rng, 2, 9), [length, length // 2], heads, max_len=length + 9)


@pytest.mark.parametrize("window", [1, 2, 5, 64, 100, 512, 5000])
@pytest.mark.parametrize("nodes", [1, 11, 64])
def test_attention_windows(dev, window, nodes):
    """Windows shorter than a branch, than the tree and than the sequence; a chain
    of nodes is the deepest tree."""
    rng = np.random.default_rng(window)
    p = random_parents(rng, 3, nodes)
    p[0] = np.arange(nodes) - 1
    check_attention(dev, p, [700, 3, 90], (8, 2, 64), window=window, max_len=800)
    check_attention(dev, p, [0, 500, 61], (4, 1, 128), window=window, max_len=800)


def test_attention_row_map_padding_and_the_caches_end(dev):
    parents = [[-1, 0, -1, 2, 5, 0, -7, 1], [-2, 0, 1, 2, 3, 4, 5, 6], [-1, 0, 1, 2, 3, 4, 5, 6], [-1] * 8]
    check_attention(dev, parents, [300, 4, 59, 1], (8, 2, 64), rows=6, row_map=[5, 0, 2, 3], max_len=400)
    check_attention(dev, parents, [30, 4, 59, 64], (8, 2, 64), max_len=64)  # nodes past the cache's end
    check_attention(dev, parents, [30, 4, 64, 64], (8, 2, 64), max_len=64, window=1)  # some of them see nothing


@pytest.mark.parametrize("heads", [(8, 1, 64), (8, 2, 128), (64, 2, 64)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_unseen_values_do_not_reach_a_node(dev, heads, bad):
    """Stale slots behind the tree, padding's slots, positions before the window and
    a sibling's rows: what a node does not see may hold anything; what it does see
    shows."""
    parents = [[-1, 0, 0, 2, -1, 1, 9], [-1, -1, -1, -1, -1, -1, -1], [-1, 0, 1, 2, 3, 4, 5]]
    seqlen = [150, 17, 200]

    def stale(k, v):
        for r, n in enumerate(seqlen):
            for i, up in enumerate(ot.branches(parents[r])):
                if up is None:
                    k[r, :, n + i] = bad
                    v[r, :, n + i] = bad
            k[r, :, n + 7:] = bad
            v[r, :, n + 7:] = bad

    check_attention(dev, parents, seqlen, heads, max_len=256, spoil=stale)

    def before(k, v):
        stale(k, v)
        for r, n in enumerate(seqlen):
            k[r, :, :max(0, n - 19)] = bad
            v[r, :, :max(0, n - 19)] = bad

    check_attention(dev, parents, seqlen, heads, max_len=256, window=20, spoil=before)

    def sibling(k, v):
        stale(k, v)
        v[0, :, 152] = bad  # node 2: seen by itself and by node 3
        v[0, 0, 151, 3] = bad  # one value of node 1: seen by itself and by node 5
        v[2, 0, 190, 5] = bad  # in the third row's sequence: seen by the nodes whose window holds it

    check_attention(dev, parents, seqlen, heads, max_len=256, spoil=sibling)
    check_attention(dev, parents, seqlen, heads, max_len=256, window=13, spoil=sibling)


def test_attention_scores_of_any_size(dev):
    """Rising scores (each chunk raises the maximum by far more than the reference
    maximum is kept within), falling ones, and very large ones."""
    from maple_amd.kernels import tree_attention

    nq, nkv, d, n, t = 8, 1, 64, 1500, 4
    parents = [[-1, 0, 1, 1]]
    q = torch.ones(1, t, nq, d, device=dev, dtype=torch.bfloat16)
    v = bf16(dev, 1, nkv, n + t, d, seed=2)
    ramp = torch.arange(n + t, device=dev, dtype=torch.float32)
    for rise in (ramp, -ramp, ramp * 4, torch.where(ramp == 700, 200.0, -200.0), torch.zeros_like(ramp)):
        k = (rise / d).to(torch.bfloat16).view(1, 1, -1, 1).expand(1, nkv, n + t, d).contiguous()
        out = tree_attention(q, k, v, torch.tensor([n], device=dev), as_parents(parents, dev), scale=0.25)
        compare_attention(out, q, k, v, parents, [n], 0.25)


@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("heads,n", [((32, 1, 64), 1500), ((16, 1, 128), 1500), ((8, 2, 64), 9)])
def test_attention_scores_past_float32s_whole_numbers(dev, heads, n, window):
    """Finite scores up to 2^120, of either sign, where a step of float32 is more than
    an exponent can hold: equal ones weigh alike, of others the largest takes all
    (scores are powers of two times small numbers: exact in bf16 and in float32, so
    equal where they are equal and far apart else)."""
    from maple_amd.kernels import tree_attention

    nq, nkv, d = heads
    t = 5
    parents = [[-1, 0, 1, 1, 3]]
    q = torch.zeros(1, t, nq, d, device=dev, dtype=torch.bfloat16)
    q[..., 0] = 1
    v = bf16(dev, 1, nkv, n + t, d, seed=2)
    at = torch.arange(n + t, device=dev, dtype=torch.float64)
    shapes = (torch.ones_like(at), -torch.ones_like(at), 1 + (at * 7 % 100 < 1), -1 - (at * 7 % 100 > 1).double(),
              (at // 16).clamp(max=100), -(at // 16).clamp(max=100), torch.where(at < n - 20, -1.0, 1.0),
              torch.where(at < n - 20, 1.0, 0.0))
    for power in (20, 27, 30, 32, 45, 113):
        for shape in shapes:
            k = bf16(dev, 1, nkv, n + t, d, seed=3)
            k[..., 0] = (shape * 2.0 ** power).to(torch.bfloat16)
            for scale in (1.0, -0.125):
                out = tree_attention(q, k, v, torch.tensor([n], device=dev), as_parents(parents, dev), scale=scale,
                                     window=window)
                compare_attention(out, q, k, v, parents, [n], scale, window)


@pytest.mark.parametrize("heads", [(32, 1, 64), (16, 1, 128), (4, 4, 64)])
def test_attention_references_that_stay_too_low(dev, heads):
    """Scores that stay above the first ones for the rest of the sequence: just
    below what moves the reference, one jump and level, level after a spike, rising
    slowly; in nats over a scale of 1, exact in bf16."""
    from maple_amd.kernels import tree_attention

    nq, nkv, d = heads
    n, t = 6000, 5
    parents = [[-1, 0, 1, 1, 3]]
    q = torch.zeros(1, t, nq, d, device=dev, dtype=torch.bfloat16)
    q[..., 0] = 1
    v = bf16(dev, 1, nkv, n + t, d, seed=2)
    at = torch.arange(n + t, device=dev)
    for rise in (torch.where(at < 40, 0.0, 10.5), torch.where(at < 64, -60.0, 0.0), torch.where(at == 200, 11.0, 0.0),
                 torch.where(at < 100, -200.0, torch.where(at == 3000, 11.0, 0.0)), (at // 500) * 4.0,
                 torch.where(at % 700 == 699, 60.0, -20.0), torch.where(at < n, -150.0, -160.0)):
        k = bf16(dev, 1, nkv, n + t, d, seed=3)
        k[..., 0] = rise.to(torch.bfloat16)
        out = tree_attention(q, k, v, torch.tensor([n], device=dev), as_parents(parents, dev), scale=1.0)
        compare_attention(out, q, k, v, parents, [n], 1.0)


@pytest.mark.parametrize("heads", [(8, 1, 64), (8, 2, 128)])
def test_attention_of_what_is_not_finite_stays_in_its_rows(dev, heads):
    """A NaN in one node's query, NaN or infinite keys that nodes do see: those rows
    as in 64 bits, every other row untouched."""
    from maple_amd.kernels import tree_attention

    nq, nkv, d = heads
    parents, seqlen = [[-1, 0, 1, 1, 0, 4], [-1, 0, 1, 2, 3, 4], [-1] * 6], [300, 290, 130]
    q = bf16(dev, 3, 6, nq, d)
    k, v = bf16(dev, 3, nkv, 320, d, seed=1), bf16(dev, 3, nkv, 320, d, seed=2)
    q[0, 3, :, 5] = float("nan")
    q[1, 2, 0, 0] = float("inf")
    k[1, 0, 40, 7] = float("nan")  # one KV head of the second row: all its nodes see it
    k[0, :, 304, 3] = float("inf")  # node 4 of the first: seen by itself and by node 5
    sl = torch.tensor(seqlen, device=dev)
    for window in (None, 280):  # (280: position 40 is seen by the second row's first nodes alone)
        out = tree_attention(q, k, v, sl, as_parents(parents, dev), scale=d ** -0.5, window=window)
        compare_attention(out, q, k, v, parents, seqlen, d ** -0.5, window)


@pytest.mark.parametrize("heads", [(8, 1, 64), (8, 2, 128)])
@pytest.mark.parametrize("n,max_len", [(0, 16), (70, 100), (2000, 2100)])
def test_attention_scores_of_minus_infinity(dev, heads, n, max_len):
    """Keys that give one head -inf everywhere: 0 there, as where a node sees
    nothing; the other heads as in 64 bits, and so the first where it meets one
    finite score."""
    from maple_amd.kernels import tree_attention

    nq, nkv, d = heads
    parents = [[-1, 0, 0, 1]]
    q = bf16(dev, 1, 4, nq, d)
    q[..., 0] = 0
    k, v = bf16(dev, 1, nkv, max_len, d, seed=1), bf16(dev, 1, nkv, max_len, d, seed=2)
    q[:, :, 0, 0], q[:, :, 1:, 0] = 1.0, 2.0 ** -100
    k[..., 0] = -3e38  # x 1 x scale: -inf in no float32, but alone in its sum
    lone = k.clone()
    k[..., 0] = float("-inf")
    sl, p = torch.tensor([n], device=dev), as_parents(parents, dev)
    out = tree_attention(q, k, v, sl, p, scale=d ** -0.5)
    assert (out == 0).all()  # (-inf for every head: 2^-100 x -inf too)
    lone[0, :, n + 1, 0] = 0  # node 1, which node 3 sees too
    k[0, :, n + 1, 0] = 0
    out = tree_attention(q, k, v, sl, p, scale=d ** -0.5)
    assert (out[:, [0, 2]] == 0).all()
    for node in (1, 3):
        for h in range(nq):
            assert torch.equal(out[0, node, h], v[0, h * nkv // nq, n + 1])
    out = tree_attention(q, lone, v, sl, p, scale=d ** -0.5)
    compare_attention(out[:, :, :1], q[:, :, :1], lone[:, :1], v[:, :1], parents, [n], d ** -0.5)
    # The other heads' scores are 2^-100 x -3e38 = -2.4e8 and the other dims' few units: a step of
    # float32 is 16 there, so those units are not held and the weights of equal keys say nothing; node 1's
    # finite key takes all where it is seen, and any weights give values between the least and the largest V.
    for node in (1, 3):
        for h in range(1, nq):
            assert torch.equal(out[0, node, h], v[0, h * nkv // nq, n + 1])
    lo, hi = (f(v[:, :, :n + 4].float(), 2).view(1, 1, nkv, 1, d) for f in (torch.amin, torch.amax))
    rest = out.float().view(1, 4, nkv, nq // nkv, d)
    assert ((rest >= lo - 2.0 ** -7 * lo.abs()) & (rest <= hi + 2.0 ** -7 * hi.abs())).all()


def test_attention_windows_past_every_distance(dev):
    """As without a window, up to the largest one."""
    from maple_amd.kernels import tree_attention

    rng = np.random.default_rng(5)
    parents = as_parents(random_parents(rng, 2, 64, ragged=False), dev)
    q, k, v = bf16(dev, 2, 64, 8, 64), bf16(dev, 2, 2, 640, 64, seed=1), bf16(dev, 2, 2, 640, 64, seed=2)
    sl = torch.tensor([576, 0], device=dev)
    want = tree_attention(q, k, v, sl, parents, scale=0.125)
    for window in (640, 641, 703, 705, 2 ** 31, 2 ** 62, 2 ** 63 - 1):
        out = tree_attention(q, k, v, sl, parents, scale=0.125, window=window)
        if window > 704:
            assert torch.equal(out, want)
        else:  # (other splits: their sums' order)
            compare_attention(out, q, k, v, parents.cpu().numpy(), [576, 0], 0.125, window)


@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30, 3.0])
def test_attention_scales(dev, scale):
    from maple_amd.kernels import tree_attention

    rng = np.random.default_rng(3)
    parents = random_parents(rng, 2, 9)
    q, k, v = bf16(dev, 2, 9, 8, 64), bf16(dev, 2, 2, 500, 64, seed=1), bf16(dev, 2, 2, 500, 64, seed=2)
    out = tree_attention(q, k, v, torch.tensor([480, 77], device=dev), as_parents(parents, dev), scale=scale)
    compare_attention(out, q, k, v, parents, [480, 77], scale)


def test_one_node_is_decode_gqa_attn(dev):
    from maple_amd.kernels import decode_gqa_attn, tree_attention

    b, nq, nkv, d, n = 4, 32, 4, 64, 700
    q, k, v = bf16(dev, b, 1, nq, d), bf16(dev, b, nkv, n, d, seed=1), bf16(dev, b, nkv, n, d, seed=2)
    sl = torch.tensor([0, 127, 500, 699], device=dev)
    one = decode_gqa_attn(q.reshape(b, nq, 1, d), k, v, sl, scale=d ** -0.5, window=None)
    two = tree_attention(q, k, v, sl, as_parents([[-1]] * b, dev), scale=d ** -0.5)
    parents, s = [[-1]] * b, sl.tolist()
    compare_attention(two, q, k, v, parents, s, d ** -0.5)
    compare_attention(one.reshape(b, 1, nq, d), q, k, v, parents, s, d ** -0.5)


def test_attention_offsets_past_32_bits(dev):
    """A cache of more than 2^32 values: a row that starts past 2^32, and positions
    past 2^31 values into one (seen through a window)."""
    nkv, d = 2, 64
    n = 17_500_000  # 2 x 17.5M x 64 = 2.24e9 values a row
    k = torch.empty(3, nkv, n, d, device=dev, dtype=torch.bfloat16)
    v = torch.empty_like(k)
    seqlen = [40, n - 30]
    for r, s in zip((2, 1), seqlen):
        for c, seed in ((k, 1), (v, 2)):
            lo = max(0, s - 70)
            c[r, :, lo:s + 12] = bf16(dev, nkv, s + 12 - lo, d, seed=seed + r)
    rng = np.random.default_rng(0)
    parents = random_parents(rng, 2, 12, ragged=False)
    from maple_amd.kernels import commit_tree, tree_attention

    q = bf16(dev, 2, 12, 8, d)
    sl, rm = torch.tensor(seqlen, device=dev), torch.tensor([2, 1], device=dev)
    out = tree_attention(q, k, v, sl, as_parents(parents, dev), scale=0.125, window=64, row_map=rm)
    for r, (cr, s) in enumerate(zip((2, 1), seqlen)):
        lo = max(0, s - 70)
        compare_attention(out[r:r + 1], q[r:r + 1], k[cr:cr + 1, :, lo:s + 12], v[cr:cr + 1, :, lo:s + 12],
                          parents[r:r + 1], [s - lo], 0.125, 64)
    want = k[1, :, n - 30 + 11].clone(), v[2, :, 40 + 7].clone()
    path = torch.full((2, 12), -1, dtype=torch.int32, device=dev)
    path[0, :2], path[1, :2] = torch.tensor([0, 7]), torch.tensor([0, 11])
    new = commit_tree([k], [v], sl, path, torch.tensor([1, 1], dtype=torch.int32, device=dev), row_map=rm)
    assert new.tolist() == [42, n - 28]
    assert torch.equal(k[1, :, n - 29], want[0]) and torch.equal(v[2, :, 41], want[1])


# ---------------------------------------------------------------------------
# Verification
# ---------------------------------------------------------------------------
def draft(dev, batch, nodes, vocab, *, seed=0, dtype=torch.bfloat16, probs=False, parents=None, spread=2.0):
    """Logits with a few likely tokens a row and a tree of them."""
    rng = np.random.default_rng(seed)
    parents = random_parents(rng, batch, nodes) if parents is None else np.asarray(parents)
    x = rng.normal(size=(batch, nodes, vocab)) * spread
    likely = rng.integers(0, vocab, size=(batch, nodes, 4))
    np.put_along_axis(x, likely, 7 + 4 * rng.random(likely.shape), axis=2)
    up = np.clip(parents, 0, nodes - 1)
    tokens = np.take_along_axis(np.take_along_axis(likely, up[:, :, None], 1), rng.integers(0, 4, (batch, nodes, 1)), 2)
    q = None
    if probs:
        y = np.take_along_axis(x, up[:, :, None], 1) + rng.normal(size=x.shape) * 0.5
        y = np.exp(y - y.max(-1, keepdims=True))
        q = torch.tensor(y / y.sum(-1, keepdims=True), device=dev, dtype=torch.float32)
        cdf = np.cumsum(np64(q), -1)
        tokens = (cdf < rng.random((batch, nodes, 1)) * cdf[..., -1:]).sum(-1, keepdims=True)
    return dict(logits=torch.tensor(x, device=dev).to(dtype), tokens=torch.tensor(tokens[..., 0], device=dev),
                parents=parents, uniform=torch.tensor(rng.random((batch, nodes)), device=dev, dtype=torch.float32),
                draft_probs=q)


def check_verify(dev, s, **kw):
    from maple_amd.kernels import verify_tree

    kw = {**dict(temperature=0.8, top_p=0.95, top_k=20), **kw}
    got = verify_tree(s["logits"], s["tokens"], as_parents(s["parents"], dev), s["uniform"],
                      draft_probs=s.get("draft_probs"), **kw)
    b, t = s["tokens"].shape
    assert got.tokens.dtype == torch.int64 and got.accepted.dtype == got.path.dtype == torch.int32
    logits, u, tok = np64(s["logits"]), np64(s["uniform"]), s["tokens"].cpu().numpy()
    q = None if s.get("draft_probs") is None else np64(s["draft_probs"])
    for r in range(b):
        out, path = ot.verify(logits[r], tok[r], s["parents"][r], u[r], probs=None if q is None else q[r], **kw)
        assert got.accepted[r].item() == len(path) - 1, r
        assert got.path[r].tolist() == path + [-1] * (t - len(path)), r
        assert got.tokens[r].tolist() == out + [-1] * (t - len(out)), r
    return got


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("top_k", [1, 2, 50, 64])
@pytest.mark.parametrize("nodes", [1, 2, 9, 64])
def test_verify_matches_the_oracle(dev, probs, top_k, nodes):
    s = draft(dev, 6, nodes, 3001, seed=nodes + top_k, probs=probs)
    for top_p in (1.0, 0.9, 0.3):
        got = check_verify(dev, s, top_k=top_k, top_p=top_p)
    if nodes > 2 and not probs:
        assert got.accepted.max().item() > 0  # (the cases do accept)


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 255, 1000, 4095, 4096, 4097, 8209, 100003])
def test_verify_vocabularies(dev, vocab):
    check_verify(dev, draft(dev, 2, 5, vocab, seed=vocab), top_k=min(vocab, 64))
    check_verify(dev, draft(dev, 2, 5, vocab, seed=vocab, probs=True), top_k=min(vocab, 7), temperature=1.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_verify_types_and_unaligned_rows(dev, dtype):
    s = draft(dev, 3, 7, 2003, dtype=dtype, probs=True)
    wide = torch.zeros(3, 9, 2003 + 13, device=dev, dtype=dtype)
    pw = torch.zeros(3, 8, 2003 + 5, device=dev, dtype=dtype)
    wide[:, 1:8, 5:2008] = s["logits"]
    pw[:, :7, 1:2004] = s["draft_probs"].to(dtype)
    s["logits"], s["draft_probs"] = wide[:, 1:8, 5:2008], pw[:, :7, 1:2004]
    check_verify(dev, s)


def test_verify_a_full_batch_of_long_rows(dev):
    """As many rows as a launch aims for and more (one segment a row), and few of
    them (many segments)."""
    for b, t in ((70, 16), (1, 1), (1, 9)):
        check_verify(dev, draft(dev, b, t, 32000, seed=b + t), top_k=64)


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few", "lowest", "minus_inf", "two_levels"])
def test_verify_ties_masks_and_orders(dev, kind):
    """Logits that tie over whole rows, arrive in the worst order for a running
    threshold, or are masked by -inf or by the type's lowest value."""
    s = draft(dev, 2, 6, 9001, seed=4)
    x = s["logits"]
    ramp = torch.arange(9001, device=dev, dtype=torch.float32)
    if kind == "equal":
        x.fill_(1.5)
    elif kind == "rising":
        x.copy_(ramp / 16)
    elif kind == "falling":
        x.copy_(-ramp / 16)
    elif kind == "few":
        x.fill_(float("-inf"))
        x[..., 100:103] = torch.tensor([1.0, 2.0, 2.0], device=dev)
    elif kind == "lowest":
        keep = x[..., 5000:5003].clone()
        x.fill_(torch.finfo(torch.bfloat16).min)
        x[..., 5000:5003] = keep
    elif kind == "minus_inf":
        x[..., ::2] = float("-inf")
    else:
        x.copy_((ramp % 3 == 0).float())
    s["tokens"][:] = torch.tensor([0, 101, 102, 5001, 0, 9000], device=dev)
    for top_k in (1, 5, 64):
        check_verify(dev, s, top_k=top_k, top_p=1.0)


def test_verify_repeated_out_of_range_and_zero_probability_tokens(dev):
    parents = [[-1, 0, 0, 0, 0, 1, 2]] * 3
    s = draft(dev, 3, 7, 500, parents=parents)
    best = s["logits"].float().argmax(-1)
    s["tokens"][0] = best[0, 0]  # every sibling the same token
    s["tokens"][1] = torch.tensor([0, -1, 500, 1 << 40, -(1 << 40), 3, 3], device=dev)
    for u in (0.0, 0.5, 0.999999):
        s["uniform"].fill_(u)
        check_verify(dev, s)
        s["draft_probs"] = torch.zeros(3, 7, 500, device=dev)  # nothing is likely: any possible token is taken
        check_verify(dev, s)
        s["draft_probs"] = torch.ones(3, 7, 500, device=dev)  # nothing is left: the law stays
        check_verify(dev, s)
        s["draft_probs"] = None


def test_verify_padding_and_rows_without_a_sequence(dev):
    parents = [[-1, 0, -1, 2, 5, 0, -7, 1], [-2, 0, 1, 2, 3, 4, 5, 6], [-1] * 8, [-1, 0, 1, 2, 3, 4, 5, 6]]
    s = draft(dev, 4, 8, 700, parents=parents, seed=2)
    for u in (0.0, 0.3):  # 0 accepts every token that is possible
        s["uniform"].fill_(u)
        check_verify(dev, s, top_k=64, top_p=1.0)


@pytest.mark.parametrize("top_k", [1, 2, 5, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_verify_infinite_logits(dev, top_k, dtype):
    """Logits of +inf (a forced token) carry all of the law, alike where there are
    several; rows of nothing but -inf weigh their top_k first tokens alike."""
    parents = [[-1, 0, 0, 1, 2], [-1, 0, 1, 2, 3], [-1, 0, 0, 0, 0], [-1, 0, 0, 0, 0]]
    s = draft(dev, 4, 5, 900, parents=parents, seed=3, dtype=dtype)
    x = s["logits"]
    x[0, 0, 700] = x[0, 2, 3] = float("inf")  # forced: node 2's token, then node 4's
    x[1, :, 899] = float("inf")  # along a chain
    x[2, 0, [11, 12, 500]] = float("inf")  # three alike
    x[3] = float("-inf")
    s["tokens"] = torch.tensor([[0, 1, 700, 5, 3], [0, 899, 899, 899, 7], [0, 13, 12, 500, 11], [0, 800, 1, 0, 2]],
                               device=dev)
    drawn = torch.zeros(4, 5, 900, device=dev)
    drawn.scatter_(2, s["tokens"].unsqueeze(-1), 0.5)
    for u in (0.0, 0.3, 0.7, 0.999999):
        s["uniform"].fill_(u)
        for top_p in (1.0, 0.55):
            s["draft_probs"] = None
            got = check_verify(dev, s, top_k=top_k, top_p=top_p)
            # a forced token that was drafted is always kept
            assert got.path[0, :3].tolist() == [0, 2, 4] and got.accepted[1] == 3 and got.tokens[1, 3] == 899
            s["draft_probs"] = drawn
            check_verify(dev, s, top_k=top_k, top_p=top_p)


def test_verify_without_a_draft_is_the_sampler(dev):
    from maple_amd.kernels.sampler import fused_sample_batched

    s = draft(dev, 40, 1, 151936, seed=1, spread=3.0)
    for kw in (dict(temperature=0.7, top_p=0.9, top_k=50), dict(temperature=1.0, top_p=1.0, top_k=1)):
        got = check_verify(dev, s, **kw)
        one = fused_sample_batched(s["logits"][:, 0], s["uniform"][:, 0], **kw)
        # (the sampler's law is float32: a uniform within 1e-6 of a border may fall to the other side)
        assert (got.tokens[:, 0] == one).float().mean() >= 0.97


# ---------------------------------------------------------------------------
# Commit
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("layers,heads", [(1, (4, 64)), (3, (2, 128)), (65, (1, 64))])
@pytest.mark.parametrize("nodes", [1, 2, 8, 64])
def test_commit_moves_the_accepted_rows(dev, layers, heads, nodes):
    from maple_amd.kernels import commit_tree

    nkv, d = heads
    rng = np.random.default_rng(nodes + layers)
    b, n = 5, 200
    ks = [bf16(dev, b + 1, nkv, n, d, seed=2 * i) for i in range(layers)]
    vs = [bf16(dev, b + 1, nkv, n, d, seed=2 * i + 1) for i in range(layers)]
    seqlen, rm = [0, 7, 100, n - nodes, n - nodes // 2], [5, 1, 0, 2, 4]
    path, acc = np.full((b, nodes), -1), np.zeros(b, np.int64)
    for r in range(b):
        m = int(rng.integers(0, nodes)) if r else nodes - 1
        path[r, :m + 1] = np.concatenate([[0], np.sort(rng.permutation(nodes - 1)[:m]) + 1])
        acc[r] = m
    acc[2], path[2] = -1, -1
    want = []
    for c in ks + vs:
        w = c.clone()
        for r in range(b):
            for j in range(1, acc[r] + 1):
                if seqlen[r] + path[r, j] < n:
                    w[rm[r], :, seqlen[r] + j] = c[rm[r], :, seqlen[r] + path[r, j]]
        want.append(w)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    sl = torch.tensor(seqlen, device=dev)
    new = commit_tree(ks, vs, sl, i32(path), i32(acc), row_map=torch.tensor(rm, device=dev))
    assert new.tolist() == [s + int(a) + 1 for s, a in zip(seqlen, acc)] and sl.tolist() == seqlen
    for got, w in zip(ks + vs, want):
        assert torch.equal(got.view(torch.int16), w.view(torch.int16))


# ---------------------------------------------------------------------------
# Trees that fit the cache
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_fit_tree_leaves_out_nodes_past_the_caches_end(dev, dtype):
    from maple_amd.kernels import fit_tree

    parents = torch.tensor([[-1, 0, 0, 1]] * 5 + [[-2, 0, 0, 1]], dtype=dtype, device=dev)
    seqlen = torch.tensor([0, 4, 6, 7, 8, 5], device=dev)
    want = [[-1, 0, 0, 1], [-1, 0, 0, 1], [-1, 0, -2, -2], [-1, -2, -2, -2], [-2] * 4, [-2, 0, 0, -2]]
    got = fit_tree(parents, seqlen, 8)
    assert got.dtype == torch.int32 and got.is_contiguous() and got.tolist() == want
    assert fit_tree(parents, seqlen, 1 << 40).tolist() == parents.tolist()
    assert fit_tree(parents, seqlen, 0).tolist() == [[-2] * 4] * 6
    wide = torch.full((6, 9), 5, dtype=dtype, device=dev)
    wide[:, 3:7] = parents
    assert fit_tree(wide[:, 3:7], seqlen.int(), 8).tolist() == want
    assert fit_tree(parents[:0], seqlen[:0], 8).shape == (0, 4)
    if dtype == torch.int64:  # no large value becomes a node
        far = torch.tensor([[-1, 1 << 32, (1 << 32) + 1, -(1 << 32)]], device=dev)
        assert fit_tree(far, seqlen[:1], 8).tolist() == [[-1, 64, 64, -2]]
        far = torch.tensor([2 ** 63 - 1, -2 ** 63], device=dev)
        assert fit_tree(parents[:2], far, 8).tolist() == [[-2] * 4, [-1, 0, 0, 1]]
    rng = np.random.default_rng(1)
    if dtype == torch.int32:  # in place, through the library
        from maple_amd import _lib

        same = parents.clone()
        _lib.call("ma_tree_fit", same.data_ptr(), 0, 6, 4, seqlen.data_ptr(), 8, same.data_ptr(), _lib.stream_of(same))
        assert same.tolist() == want
    for b, t in ((1, 64), (1023, 64), (300, 7), (65535, 1)):
        p = torch.tensor(random_parents(rng, min(b, 40), t), dtype=dtype, device=dev).repeat(-(-b // min(b, 40)), 1)[:b]
        sl = torch.tensor(rng.integers(0, 200, b), device=dev)
        fits = sl[:, None] + torch.arange(t, device=dev) < 130
        assert torch.equal(fit_tree(p, sl, 130), torch.where(fits, p, -2).int())


# ---------------------------------------------------------------------------
# Streams and graphs
# ---------------------------------------------------------------------------
def _step(k, v, s, heads, cos, sin, qkv, rot, window=None):
    from maple_amd.kernels import apply_qkv_tree, commit_tree, tree_attention, verify_tree

    nq, nkv, d = heads
    q = apply_qkv_tree(qkv, None, None, cos, sin, k, v, s["seqlen"], s["parents"], num_heads=nq, num_kv_heads=nkv,
                       head_dim=d, rotary_dim=rot)
    out = tree_attention(q, k, v, s["seqlen"], s["parents"], scale=d ** -0.5, window=window)
    ver = verify_tree(s["logits"], s["tokens"], s["parents"], s["uniform"], temperature=0.8, top_p=0.95, top_k=50,
                      draft_probs=s["draft_probs"])
    new = commit_tree([k], [v], s["seqlen"], ver.path, ver.accepted)
    return (q, out, *ver, new, k, v)


def _step_inputs(dev, seed, b=3, t=12, heads=(8, 2, 64), n=600):
    s = draft(dev, b, t, 5000, seed=seed, probs=True)
    s["parents"] = as_parents(s["parents"], dev)
    rng = np.random.default_rng(seed)
    s["seqlen"] = torch.tensor(rng.integers(0, n - t, b), device=dev)
    nq, nkv, d = heads
    return s, bf16(dev, b, nkv, n, d, seed=seed), bf16(dev, b, nkv, n, d, seed=seed + 1), bf16(
        dev, b, t, (nq + 2 * nkv) * d, seed=seed + 2)


def test_a_run_of_them_captured_and_replayed(dev):
    """Two graphs of the whole run captured on one stream and replayed in turn on
    new inputs, with eager work between: every replay equals the eager run."""
    heads, rot = (8, 2, 64), 32
    cos, sin = tables(700, rot, dev)
    graphs = []
    side = torch.cuda.Stream()
    for seed in (1, 2):
        s, k, v, qkv = _step_inputs(dev, seed)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(k, v, s, heads, cos, sin, qkv, rot)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = _step(k, v, s, heads, cos, sin, qkv, rot)
        torch.cuda.current_stream().wait_stream(side)
        graphs.append((g, s, k, v, qkv, out))
    for rep in range(4):
        for i, (g, s, k, v, qkv, out) in enumerate(graphs):
            n, nk, nv, nqkv = _step_inputs(dev, 100 + 2 * rep + i)
            want = [x.clone() for x in _step(nk.clone(), nv.clone(), n, heads, cos, sin, nqkv, rot)]
            for name in ("logits", "tokens", "parents", "uniform", "draft_probs", "seqlen"):
                s[name].copy_(n[name])
            k.copy_(nk), v.copy_(nv), qkv.copy_(nqkv)
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b), (rep, i)


def test_runs_on_two_streams_at_once(dev):
    heads, rot = (8, 2, 64), 32
    cos, sin = tables(700, rot, dev)
    sets = [_step_inputs(dev, seed) for seed in (5, 6)]
    want = [[x.clone() for x in _step(k.clone(), v.clone(), s, heads, cos, sin, qkv, rot)] for s, k, v, qkv in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for st, (s, k, v, qkv) in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(_step(k.clone(), v.clone(), s, heads, cos, sin, qkv, rot))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_same_bits_again(dev):
    heads, rot = (32, 4, 64), 32
    cos, sin = tables(4300, rot, dev)
    s, k, v, qkv = _step_inputs(dev, 9, b=2, t=32, heads=heads, n=4200)
    first = [x.clone() for x in _step(k.clone(), v.clone(), s, heads, cos, sin, qkv, rot)]
    for _ in range(3):
        again = _step(k.clone(), v.clone(), s, heads, cos, sin, qkv, rot)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
