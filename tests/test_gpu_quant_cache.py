"""Quantised caches and shared prefixes (kernels/quant_cache.py) against the float64
oracle (oracle/quant_cache.py).

Tolerances.  Codes and scales of bf16 values are exact: scaling by a power of two
is, and the nearest code is one.  QKV: q is rounded to bf16 once (2^-8 of its value)
and the float32 norm and rotation are within 2^-16 of the sum of the terms'
magnitudes; K's codes are those of the bf16 K that ``apply_qkv_tree`` stores for one
node, to the bit (the same arithmetic), and V's those of V.  Attention: each
weight p is rounded to bf16 (2^-8 of it) in the numerator and, alike, in the sum, so the
quotient is off by at most 2 x 2^-8 of sum p |v|, its rounding adds 2^-8 of the output,
and float32 scores, exponentials and sums stay within 2^-12 of sum p |v| at these
score sizes (scores of up to 2^5, each within 2^-17, and another 2^-14 where the parts
of a sequence are joined)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import quant_cache as oq
from oracle import tree as ot

pytestmark = pytest.mark.gpu

EPS = 1e-6


def np64(t):
    return t.detach().double().cpu().numpy()


def bf16(dev, *shape, seed=0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16)


def exps(scale):
    return scale.view(torch.uint8).cpu().numpy().astype(np.int64) - 127


def i64(dev, x):
    return None if x is None else torch.tensor(x, device=dev, dtype=torch.int64)


def filled(dev, rows, nkv, n, d, seed=0):
    """A quantised cache of random values."""
    from maple_amd.kernels import make_quant_kv, quantize_kv

    c = make_quant_kv(rows, nkv, n, d, dev)
    k, v = bf16(dev, rows, nkv, n, d, seed=seed), bf16(dev, rows, nkv, n, d, seed=seed + 1)
    return quantize_kv(k, v * torch.exp2(torch.arange(n, device=dev) % 5 - 2).view(1, 1, n, 1).bfloat16(), c)


def values(cache):
    """A cache's K and V in float64."""
    if len(cache) == 2:
        return np64(cache[0]), np64(cache[1])
    return tuple(oq.decode(np64(c), exps(s)) for c, s in ((cache[0], cache[2]), (cache[1], cache[3])))


def bits(cache):
    return [t.view(torch.uint8 if t.element_size() == 1 else torch.int16).clone() for t in cache]


# ---------------------------------------------------------------------------
# Prompts in, and back
# ---------------------------------------------------------------------------
def check_quantize(dev, k, v, *, max_len, start=None, lengths=None, rows=None, row_map=None):
    from maple_amd.kernels import quantize_kv

    b, nkv, t, d = k.shape
    cache = filled(dev, rows or b, nkv, max_len, d, seed=91)
    before = bits(cache)
    assert quantize_kv(k, v, cache, start=i64(dev, start), lengths=i64(dev, lengths), row_map=i64(dev, row_map)) is cache
    left = np.ones((rows or b, max_len), bool)
    for x, codes, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        want_c, want_e = oq.encode(np64(x))
        got_c, got_e = np64(codes), exps(scale)
        for r in range(b):
            cr, s0 = r if row_map is None else row_map[r], 0 if start is None else start[r]
            n = t if lengths is None else max(0, min(t, lengths[r]))
            for i in range(n):
                if 0 <= s0 + i < max_len:
                    np.testing.assert_array_equal(got_c[cr, :, s0 + i], want_c[r, :, i])
                    assert (got_e[cr, :, s0 + i] == want_e[r, :, i]).all()
                    left[cr, s0 + i] = False
    mask = torch.tensor(left, device=dev).unsqueeze(1).expand(-1, nkv, -1)
    for now, was in zip(bits(cache), before):
        assert torch.equal(now[mask], was[mask])
    return cache


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", [1, 7, 64, 129])
def test_quantize_lengths(dev, d, t):
    check_quantize(dev, bf16(dev, 3, 4, t, d, seed=1), bf16(dev, 3, 4, t, d, seed=2), max_len=t + 5)


@pytest.mark.parametrize("d", [64, 128])
def test_quantize_strides(dev, d):
    x = bf16(dev, 2, 9, 3, d, seed=3)  # positions before heads
    check_quantize(dev, x.transpose(1, 2), x.flip(1).transpose(1, 2), max_len=12)
    y = bf16(dev, 2, 9, 3 * d + 3, seed=4)  # odd rows: no 16-byte loads
    k = y[..., 3:].unflatten(-1, (3, d))
    check_quantize(dev, k.transpose(1, 2), k.transpose(1, 2), max_len=9)
    one = bf16(dev, 1, 1, 9, d, seed=5)  # broadcast heads and rows
    check_quantize(dev, one.expand(2, 3, 9, d), one.expand(2, 3, 9, d), max_len=9)


def test_quantize_ragged_places(dev):
    k, v = bf16(dev, 4, 2, 40, 64, seed=6), bf16(dev, 4, 2, 40, 64, seed=7)
    check_quantize(dev, k, v, max_len=50, start=[0, 3, 45, 2 ** 40], lengths=[40, 17, 40, 40])
    check_quantize(dev, k, v, max_len=50, start=[-5, 0, 10, -2 ** 40], lengths=[40, 0, 99, -3])
    check_quantize(dev, k, v, max_len=41, rows=7, row_map=[6, 0, 3, 1])


@pytest.mark.parametrize("d", [64, 128])
def test_quantize_values_of_every_size(dev, d):
    rows = []
    g = np.random.default_rng(8)
    for s in range(-140, 128, 3):
        rows.append(g.normal(size=d) * 2.0 ** s)
    for s in (-126, -20, 0, 8, 100, 119, 120):  # the largest at and around the border of a power
        for m in (1.734375, 1.75, 1.7578125, 1.9921875):
            r = g.normal(size=d) * 2.0 ** (s - 3)
            r[g.integers(d)] = m * 2.0 ** min(s + 8, 127)
            rows.append(r)
    rows += [np.zeros(d), np.full(d, -0.0), np.full(d, 3.3895313892515355e38)]
    codes = np.arange(-16, 17) * 0.5 * 2.0 ** -9  # ties between subnormal codes beside a large value
    r = np.resize(codes, d)
    r[0] = 448.0
    rows.append(r)
    x = torch.tensor(np.stack(rows)).clamp(-3.3895313892515355e38, 3.3895313892515355e38).bfloat16().to(dev)
    x = x.view(1, 1, -1, d)
    check_quantize(dev, x, -x, max_len=x.shape[2])


def test_quantize_not_finite(dev):
    k = bf16(dev, 1, 2, 6, 64, seed=9)
    k[0, 0, 0, 5], k[0, 0, 1, 63], k[0, 1, 2, 0] = float("inf"), float("nan"), float("-inf")
    k[0, 1, 3] = float("nan")
    c = check_quantize(dev, k, k.flip(3), max_len=6)
    assert torch.isfinite(c.k.float()).sum() == k.numel() - 3 - 64


@pytest.mark.parametrize("d", [64, 128])
def test_dequantize(dev, d):
    from maple_amd.kernels import dequantize_kv

    c = filled(dev, 5, 3, 77, d, seed=10)
    k, v = values(c)
    for n in (77, 1, 33, 0):
        out = dequantize_kv(c, n)
        assert out.k.shape == (5, 3, n, d) and out.k.dtype == torch.bfloat16
        assert (np64(out.k) == k[:, :, :n]).all() and (np64(out.v) == v[:, :, :n]).all()
    assert torch.equal(dequantize_kv(c).k, dequantize_kv(c, 77).k)
    some = dequantize_kv(c, 50, row_map=i64(dev, [4, 4, 0]))
    assert (np64(some.k) == k[[4, 4, 0], :, :50]).all() and (np64(some.v) == v[[4, 4, 0], :, :50]).all()


@pytest.mark.parametrize("s", [-126, -60, 0, 118])
def test_round_trip_is_exact_at_any_scale(dev, s):
    """What one round trip gives, a second leaves alone (its codes are bf16 values)."""
    from maple_amd.kernels import dequantize_kv, make_quant_kv, quantize_kv

    x = (bf16(dev, 1, 2, 50, 64, seed=11).double() * 2.0 ** s).bfloat16()
    a = quantize_kv(x, x, make_quant_kv(1, 2, 50, 64, dev))
    y = dequantize_kv(a)
    if s > -100:  # (below, a code's value may need more than bf16's least step)
        b = quantize_kv(y.k, y.v, make_quant_kv(1, 2, 50, 64, dev))
        z = dequantize_kv(b)
        assert torch.equal(z.k, y.k) and torch.equal(z.v, y.v)
    ref = oq.decode(*oq.encode(np64(x)))
    assert (np.abs(np64(y.k) - ref) <= 2.0 ** -134).all()


# ---------------------------------------------------------------------------
# QKV
# ---------------------------------------------------------------------------
def tables(n, rot, dev, dtype=torch.float32):
    from maple_amd.model import rope_tables

    cos, sin = rope_tables(n, rot, 10000.0, dev)
    return cos.to(dtype), sin.to(dtype)


def check_qkv(dev, seqlen, heads, rot, *, positions=None, norm=True, max_len=64, rows=None, row_map=None,
              table=torch.float32, w_dtype=torch.float32, qkv=None, seed=0, n_pos=None):
    from maple_amd.kernels import apply_qkv_quant, apply_qkv_tree

    nq, nkv, d = heads
    b = len(seqlen)
    if qkv is None:
        qkv = bf16(dev, b, (nq + 2 * nkv) * d, seed=seed)
    cache = filled(dev, rows or b, nkv, max_len, d, seed=seed + 1)
    before = bits(cache)
    qw = kw = None
    if norm:
        qw, kw = ((torch.rand(d, device=dev) + 0.5).to(w_dtype) for _ in range(2))
    cos, sin = tables(n_pos or max_len + 64, max(rot, 2), dev, table)
    q = apply_qkv_quant(qkv, qw, kw, cos, sin, cache, i64(dev, seqlen), positions=i64(dev, positions),
                        row_map=i64(dev, row_map), num_heads=nq, num_kv_heads=nkv, head_dim=d, rotary_dim=rot,
                        use_rope=rot > 0, eps=EPS)
    assert q.shape == (b, nq, 1, d) and q.dtype == torch.bfloat16
    # the bf16 K that one tree node stores at the same position
    at = [min(max(p, 0), cos.shape[0] - 1) for p in (seqlen if positions is None else positions)]
    deep = cos.shape[0] + 1
    k16, v16 = (torch.zeros(b, nkv, deep, d, device=dev, dtype=torch.bfloat16) for _ in range(2))
    q16 = apply_qkv_tree(qkv.unsqueeze(1), qw, kw, cos, sin, k16, v16, i64(dev, at),
                         torch.full((b, 1), -1, device=dev, dtype=torch.int32), num_heads=nq, num_kv_heads=nkv,
                         head_dim=d, rotary_dim=rot, use_rope=rot > 0, eps=EPS)
    k16, v16, x = np64(k16), np64(v16), np64(qkv).reshape(b, nq + 2 * nkv, d)
    qo, c_np, s_np = np64(q), np64(cos), np64(sin)
    codes = [(np64(cache.k), exps(cache.k_scale)), (np64(cache.v), exps(cache.v_scale))]
    left = np.ones((rows or b, max_len), bool)
    for r in range(b):
        if seqlen[r] < 0:
            assert (qo[r] == 0).all()
            continue
        assert torch.equal(q[r, :, 0], q16[r, 0])
        for h in range(nq):
            ref, mag = ot.head(x[r, h], None if qw is None else np64(qw), c_np[at[r]], s_np[at[r]], rot, False, EPS)
            assert (np.abs(qo[r, h, 0] - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -16 * mag + 1e-30).all()
        if seqlen[r] >= max_len:
            continue
        cr = r if row_map is None else row_map[r]
        left[cr, seqlen[r]] = False
        for (c, e), new in zip(codes, (k16[r, :, at[r]], v16[r, :, at[r]])):
            want_c, want_e = oq.encode(new)
            np.testing.assert_array_equal(c[cr, :, seqlen[r]], want_c)
            assert (e[cr, :, seqlen[r]] == want_e).all()
    mask = torch.tensor(left, device=dev).unsqueeze(1).expand(-1, nkv, -1)
    for now, was in zip(bits(cache), before):
        assert torch.equal(now[mask], was[mask])


@pytest.mark.parametrize("heads", [(32, 4, 64), (16, 4, 128), (3, 1, 64), (2, 2, 128)])
@pytest.mark.parametrize("rot", [0, 2, 20, 32, 64])
def test_qkv_layouts_and_rotary_dims(dev, heads, rot):
    check_qkv(dev, [0, 5, 63], heads, rot)


@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("w_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_qkv_dtypes(dev, table, w_dtype):
    check_qkv(dev, [7, 1], (8, 2, 128), 128, table=table, w_dtype=w_dtype)


def test_qkv_rows_positions_and_places(dev):
    check_qkv(dev, [-1, 3, 64, 2 ** 40, -2 ** 40, 63], (4, 2, 64), 64)  # no token; behind the cache's end
    check_qkv(dev, [3, 9], (4, 2, 64), 32, positions=[100, 70])
    check_qkv(dev, [3, 9, 0], (4, 2, 64), 32, positions=[-4, 2 ** 40, 5], n_pos=20)
    check_qkv(dev, [3, 9, 11], (4, 1, 128), 64, rows=5, row_map=[4, 0, 2])
    check_qkv(dev, [3], (4, 1, 128), 64, norm=False)
    check_qkv(dev, list(range(300)), (8, 1, 64), 64, max_len=301)


def test_qkv_odd_rows(dev):
    w = (4 + 2 * 2) * 64
    qkv = bf16(dev, 3, w + 5, seed=12)
    check_qkv(dev, [1, 2, 3], (4, 2, 64), 64, qkv=qkv[:, 5:])
    check_qkv(dev, [1, 2, 3], (4, 2, 64), 64, qkv=bf16(dev, 3, w + 8, seed=13)[:, :w])


def test_qkv_not_finite_stays_in_its_head(dev):
    from maple_amd.kernels import apply_qkv_quant

    qkv = bf16(dev, 2, 8 * 64, seed=14)
    qkv[0, 4 * 64 + 3] = float("nan")  # row 0, K head 0
    qkv[1, 7 * 64 + 9] = float("inf")  # row 1, V head 1
    c = filled(dev, 2, 2, 8, 64)
    cos, sin = tables(8, 64, dev)
    w = torch.ones(64, device=dev)
    apply_qkv_quant(qkv, w, w, cos, sin, c, i64(dev, [2, 2]), num_heads=4, num_kv_heads=2, head_dim=64, rotary_dim=64)
    k, v = c.k.float()[:, :, 2], c.v.float()[:, :, 2]
    assert torch.isnan(k[0, 0]).all() and torch.isfinite(k[0, 1]).all() and torch.isfinite(k[1]).all()
    assert torch.isnan(v[1, 1]).sum() == 1 and torch.isfinite(v[0]).all() and torch.isfinite(v[1, 0]).all()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def within(got, ref, mag):
    bound = 2.0 ** -8 * np.abs(ref) + (2.0 ** -7 + 2.0 ** -12) * mag + 1e-30
    assert np.isfinite(got).all()
    worst = np.max(np.abs(got - ref) / bound)
    assert worst <= 1.0, worst


def check_attn(dev, cache, seqlen, nq, *, prefix=None, window=None, row_map=None, scale=None, q=None, seed=20):
    from maple_amd.kernels import SharedPrefix, prefix_gqa_attn, quant_gqa_attn

    rows, nkv, max_len, d = cache.k.shape
    b = len(seqlen)
    scale = d ** -0.5 if scale is None else scale
    if q is None:
        q = bf16(dev, b, nq, 1, d, seed=seed)
    kw = dict(row_map=i64(dev, row_map), scale=scale, window=window)
    if prefix is None:
        outs = [quant_gqa_attn(q, cache, i64(dev, seqlen), **kw)]
        of, plen = [-1] * b, []
    else:  # (as the sizes decide, by each row, and once for all rows)
        shared, plen, of = prefix
        forms = (None, False, True) if len(plen) <= 64 and (window or 2 ** 60) >= 2 ** 60 else (None, False)
        outs = [prefix_gqa_attn(q, cache, i64(dev, seqlen), SharedPrefix(shared, i64(dev, plen), i64(dev, of)), once=once, **kw)
                for once in forms]
        sk, sv = values(shared)
    k, v = values(cache)
    qn = np64(q)[:, :, 0]
    for r in range(b):
        cr = r if row_map is None else row_map[r]
        has = 0 <= of[r] < len(plen)
        pre, n_pre = ((sk[of[r]], sv[of[r]]), min(max(plen[of[r]], 0), sk.shape[2])) if has else (None, 0)
        ks, vs = oq.sequence((k[cr], v[cr]), min(seqlen[r] + 1, max_len), pre, n_pre, window)
        ref = oq.attend(qn[r], ks, vs, scale)
        for out in outs:
            assert out.shape == q.shape and out.dtype == torch.bfloat16
            within(np64(out[r])[:, 0], *ref)
    return outs[-1]


HEADS = [(32, 4, 64), (16, 4, 128), (16, 1, 64), (3, 1, 128), (2, 2, 64), (12, 4, 128)]


@pytest.mark.parametrize("heads", HEADS)
def test_attn_layouts(dev, heads):
    nq, nkv, d = heads
    check_attn(dev, filled(dev, 3, nkv, 300, d, seed=21), [0, 299, 150], nq)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [None, 1, 31, 64, 500, 2 ** 62, 2 ** 80])
def test_attn_lengths_and_windows(dev, d, window):
    n = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 640]
    check_attn(dev, filled(dev, len(n), 2, 640, d, seed=22), [x - 1 for x in n], 8, window=window)


@pytest.mark.parametrize("heads,n", [((8, 1, 64), 5000), ((16, 4, 128), 3001), ((8, 2, 64), 20000)])
def test_attn_long(dev, heads, n):
    nq, nkv, d = heads
    check_attn(dev, filled(dev, 2, nkv, n, d, seed=23), [n - 1, n // 3], nq)


def test_attn_many_rows(dev):
    seqlen = [(37 * i) % 90 - 1 for i in range(300)]  # some without a token
    check_attn(dev, filled(dev, 300, 1, 90, 64, seed=24), seqlen, 8)


def test_attn_rows_without_tokens_and_past_the_end(dev):
    c = filled(dev, 4, 2, 70, 128, seed=25)
    out = check_attn(dev, c, [-1, -2 ** 40, 69, 2 ** 40], 4)
    assert (out[:2] == 0).all()


def test_attn_the_most_rows(dev):
    """As many (row, KV head) pairs as a launch takes, all over two cache rows: each as the two alone."""
    from maple_amd.kernels import SharedPrefix, prefix_gqa_attn, quant_gqa_attn

    c, n = filled(dev, 2, 4, 40, 64, seed=37), 16383
    two = bf16(dev, 2, 8, 1, 64, seed=38)
    q = two.repeat(n // 2 + 1, 1, 1, 1)[:n]
    rm = torch.arange(n, device=dev) % 2
    sl = torch.full((n,), 39, device=dev)
    want = quant_gqa_attn(two, c, i64(dev, [39, 39]), scale=0.125)
    got = quant_gqa_attn(q, c, sl, row_map=rm, scale=0.125)
    assert torch.equal(got, want.repeat(n // 2 + 1, 1, 1, 1)[:n])
    pre = filled(dev, 1, 4, 50, 64, seed=39)
    for once in (False, True):
        one = [prefix_gqa_attn(x, c, y, SharedPrefix(pre, i64(dev, [50]), torch.zeros_like(y)), row_map=z, scale=0.125, once=once)
               for x, y, z in ((two, sl[:2], rm[:2]), (q, sl, rm))]
        assert torch.equal(one[1], one[0].repeat(n // 2 + 1, 1, 1, 1)[:n])


def test_attn_row_map(dev):
    c = filled(dev, 6, 2, 200, 64, seed=26)
    check_attn(dev, c, [10, 199, 64], 4, row_map=[5, 0, 5])


def poison(cache, row, lo, hi):
    """NaN codes under a NaN scale, or NaN, in a row's positions."""
    if len(cache) == 4:
        for t in cache[:2]:
            t.view(torch.uint8)[row, :, lo:hi] = 0x7F
        for t in cache[2:]:
            t.view(torch.uint8)[row, :, lo:hi] = 255
    else:
        for t in cache:
            t[row, :, lo:hi] = float("nan")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [None, 40])
def test_attn_what_is_not_seen_does_not_matter(dev, d, window):
    n = [1, 33, 64, 100, 129]
    c = filled(dev, len(n), 2, 200, d, seed=27)
    want = check_attn(dev, c, [x - 1 for x in n], 8, window=window)
    for r, x in enumerate(n):
        poison(c, r, x, 200)
        if window:
            poison(c, r, 0, max(0, x - window))
    from maple_amd.kernels import quant_gqa_attn

    got = quant_gqa_attn(bf16(dev, len(n), 8, 1, d, seed=20), c, i64(dev, [x - 1 for x in n]), scale=d ** -0.5,
                         window=window)
    assert torch.equal(got, want)


def test_attn_what_is_not_finite_and_seen_does(dev):
    from maple_amd.kernels import quant_gqa_attn

    c = filled(dev, 2, 2, 100, 64, seed=28)
    poison(c, 0, 50, 51)
    out = quant_gqa_attn(bf16(dev, 2, 4, 1, 64), c, i64(dev, [99, 99]), scale=0.125)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at", ["own", "prefix"])
@pytest.mark.parametrize("once", [False, True])
def test_attn_infinite_values(dev, d, at, once):
    """An infinite V, at the last position of a tile that is not full, is infinite in its dim and leaves the others."""
    from maple_amd.kernels import KV, SharedPrefix, prefix_gqa_attn

    own = KV(bf16(dev, 2, 2, 50, d, seed=30), bf16(dev, 2, 2, 50, d, seed=31))
    pre = KV(bf16(dev, 1, 2, 75, d, seed=32), bf16(dev, 1, 2, 75, d, seed=33))
    (own.v[0, :, 49] if at == "own" else pre.v[0, :, 74])[:, 5] = float("inf")
    out = prefix_gqa_attn(bf16(dev, 2, 4, 1, d), own, i64(dev, [49, 20]),
                          SharedPrefix(pre, i64(dev, [75]), i64(dev, [0, -1])), scale=d ** -0.5, once=once)
    assert (out[0, :, 0, 5] == float("inf")).all()
    out[0, :, 0, 5] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30, 2.0])
def test_attn_scales(dev, scale):
    # (at scale 2 scores reach 2^6.5 and their float32 errors 2^-15 of a weight: inside 2^-12)
    check_attn(dev, filled(dev, 3, 2, 150, 64, seed=29), [149, 70, 0], 8, scale=scale)


@pytest.mark.parametrize("big", [2.0 ** 20, 2.0 ** 60, 2.0 ** 110])
def test_attn_scores_of_any_size(dev, big):
    """One key far above the rest: its value is the output, at any size of the scores."""
    c = filled(dev, 1, 1, 400, 64, seed=30)
    at, q = 217, torch.zeros(1, 4, 1, 64, device=dev, dtype=torch.bfloat16)
    k = torch.zeros(1, 1, 400, 64, device=dev, dtype=torch.bfloat16)
    k[..., 0] = 1.0
    k[0, 0, at, 0] = 1.5
    from maple_amd.kernels import quant_gqa_attn, quantize_kv

    v = bf16(dev, 1, 1, 400, 64, seed=31)
    quantize_kv(k, v, c)
    q[..., 0] = big
    out = quant_gqa_attn(q, c, i64(dev, [399]), scale=1.0)
    want = values(c)[1][0, 0, at]
    assert (np.abs(np64(out)[0, :, 0] - want) <= 2.0 ** -8 * np.abs(want)).all()


def test_attn_q_strides(dev):
    c = filled(dev, 2, 2, 90, 64, seed=32)
    q = bf16(dev, 2, 8, 1, 2 * 64, seed=33)[..., 64:]
    check_attn(dev, c, [89, 40], 8, q=q)


def test_attn_offsets_past_32_bits(dev):
    """Codes of more than 2^32 bytes: rows at both ends."""
    rows, nkv, n, d = 33, 4, 2 ** 19, 64
    from maple_amd.kernels import QuantKV, dequantize_kv, quantize_kv

    k, v = (torch.zeros(rows, nkv, n, d, device=dev, dtype=torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.full((rows, nkv, n), 1, device=dev, dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2))
    c = QuantKV(k, v, ks, vs)
    x, y = bf16(dev, 2, nkv, 300, d, seed=34), bf16(dev, 2, nkv, 300, d, seed=35)
    rm = i64(dev, [rows - 1, 0])
    quantize_kv(x, y, c, start=i64(dev, [n - 300, 5]), row_map=rm)
    small = filled(dev, 2, nkv, 300, d)
    quantize_kv(x, y, small)
    got = dequantize_kv(QuantKV(*(t[rows - 1:, :, n - 300:].contiguous() for t in c)))
    assert torch.equal(got.k[0], dequantize_kv(small).k[0])
    q = bf16(dev, 1, 8, 1, d, seed=36)
    from maple_amd.kernels import quant_gqa_attn

    a = quant_gqa_attn(q, c, i64(dev, [n - 1]), row_map=rm[:1], scale=0.125, window=300)
    b = quant_gqa_attn(q, QuantKV(*(t[:1] for t in small)), i64(dev, [299]), scale=0.125)
    want, mag = oq.attend(np64(q)[0, :, 0], *(t[0] for t in values(small)), 0.125)
    within(np64(a)[0, :, 0], want, mag)
    within(np64(b)[0, :, 0], want, mag)


# ---------------------------------------------------------------------------
# Shared prefixes
# ---------------------------------------------------------------------------
def make(dev, quant, rows, nkv, n, d, seed):
    from maple_amd.kernels import KV

    if quant:
        return filled(dev, rows, nkv, n, d, seed=seed)
    return KV(bf16(dev, rows, nkv, n, d, seed=seed), bf16(dev, rows, nkv, n, d, seed=seed + 1))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("heads", HEADS)
def test_prefix_layouts(dev, quant, heads):
    nq, nkv, d = heads
    check_attn(dev, make(dev, quant, 5, nkv, 40, d, 40), [0, 39, 12, 7, -1], nq,
               prefix=(make(dev, quant, 2, nkv, 333, d, 42), [333, 100], [0, 1, 0, -1, 1]))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("plen", [0, 1, 31, 32, 33, 63, 64, 65, 129, 1000])
def test_prefix_lengths(dev, quant, d, plen):
    check_attn(dev, make(dev, quant, 4, 2, 70, d, 44), [-1, 0, 69, 33], 8,
               prefix=(make(dev, quant, 2, 2, 1000, d, 46), [plen, 1000 - plen], [0, 0, 0, 1]))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("window", [1, 50, 100, 400, 2 ** 62])
def test_prefix_windows(dev, quant, window):
    check_attn(dev, make(dev, quant, 6, 2, 130, 64, 48), [-1, 0, 129, 33, 99, 100], 8, window=window,
               prefix=(make(dev, quant, 2, 2, 300, 64, 50), [300, 77], [0, 0, 0, 1, -1, 1]))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("nq,nkv", [(2, 2), (16, 1), (6, 2)])
def test_prefix_many_rows(dev, quant, nq, nkv):
    """More rows than a workgroup's threads, prefixes with many and with no rows, indexes that name none."""
    g = np.random.default_rng(5)
    of = [int(x) for x in g.choice([0, 0, 0, 2, 4, 5, -1, 7, 2 ** 40, -2 ** 40], 333)]
    seqlen = [int(x) for x in g.integers(-1, 9, 333)]
    check_attn(dev, make(dev, quant, 333, nkv, 9, 64, 52), seqlen, nq,
               prefix=(make(dev, quant, 6, nkv, 90, 64, 54), [90, 1, 40, 7, 2 ** 40, -5], of))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("prefixes", [64, 65, 130])
def test_prefix_many_prefixes(dev, quant, prefixes):
    """As many as are read once for all of their rows, and more, which each row reads with its own positions."""
    g = np.random.default_rng(prefixes)
    of = [int(x) for x in g.integers(-1, prefixes + 1, 150)] + [prefixes - 1, 0]
    seqlen = [int(x) for x in g.integers(-1, 40, 152)]
    check_attn(dev, make(dev, quant, 152, 2, 40, 64, 55), seqlen, 4,
               prefix=(make(dev, quant, prefixes, 2, 77, 64, 57), [int(x) for x in g.integers(0, 78, prefixes)], of))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("once", [False, True])
@pytest.mark.parametrize("big", [2.0 ** 20, -2.0 ** 40, 2.0 ** 60, 2.0 ** 110])
def test_prefix_scores_of_any_size(dev, quant, once, big):
    """One key of the prefix far above the rest: its value is the output, at any size of the scores and for q of either sign."""
    from maple_amd.kernels import KV, SharedPrefix, make_quant_kv, prefix_gqa_attn, quantize_kv

    sign = 1.0 if big > 0 else -1.0
    k = torch.full((1, 1, 400, 64), 0.0, device=dev, dtype=torch.bfloat16)
    k[..., 0] = sign
    k[0, 0, 217, 0] = 1.5 * sign
    v = bf16(dev, 1, 1, 400, 64, seed=59)
    pre = quantize_kv(k, v, make_quant_kv(1, 1, 400, 64, dev)) if quant else KV(k, v)
    own = make(dev, quant, 3, 1, 30, 64, 60)
    for t in (own.k,):  # (the rows' own keys are far below)
        t.view(torch.uint8).zero_()
    q = torch.zeros(3, 16, 1, 64, device=dev, dtype=torch.bfloat16)
    q[..., 0] = big
    out = prefix_gqa_attn(q, own, i64(dev, [29, -1, 4]), SharedPrefix(pre, i64(dev, [400]), i64(dev, [0, 0, 0])), scale=1.0,
                          once=once)
    want = values(pre)[1][0, 0, 217]
    assert (np.abs(np64(out)[:, :, 0] - want) <= 2.0 ** -8 * np.abs(want)).all()


def test_prefix_long_and_split(dev):
    check_attn(dev, make(dev, True, 9, 1, 50, 64, 56), [49, 3, 7, 0, 1, 2, 20, 30, 40], 8,
               prefix=(make(dev, True, 1, 1, 9000, 64, 58), [8999], [0] * 9))
    check_attn(dev, make(dev, False, 3, 2, 50, 128, 60), [49, 3, 7], 8,
               prefix=(make(dev, False, 1, 2, 5000, 128, 62), [4801], [0] * 3))


def test_prefix_forms_by_size(dev):
    """A prefix cache past the sizes from which it is read once (rows' and prefixes' splits, tiles and one merge)."""
    check_attn(dev, make(dev, True, 32, 4, 40, 64, 61), [i % 41 - 1 for i in range(32)], 32,
               prefix=(make(dev, True, 2, 4, 2100, 64, 62), [2100, 1777], [(i % 5) // 2 for i in range(32)]))
    check_attn(dev, make(dev, False, 24, 4, 40, 128, 63), [i % 41 - 1 for i in range(24)], 16,
               prefix=(make(dev, False, 1, 4, 1100, 128, 64), [1100], [0] * 23 + [-1]))


def test_prefix_row_map(dev):
    check_attn(dev, make(dev, True, 7, 2, 60, 64, 64), [59, 3, 30], 8, row_map=[6, 0, 2],
               prefix=(make(dev, True, 2, 2, 200, 64, 66), [200, 150], [1, 0, 1]))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("once", [False, True])
def test_prefix_what_is_not_seen_does_not_matter(dev, quant, once):
    from maple_amd.kernels import SharedPrefix, prefix_gqa_attn

    own, pre = make(dev, quant, 4, 2, 70, 64, 68), make(dev, quant, 3, 2, 200, 64, 70)
    seqlen, plen, of = [-1, 10, 69, 31], [100, 64, 200], [0, 1, 0, -1]
    want = prefix_gqa_attn(bf16(dev, 4, 8, 1, 64, seed=20), own, i64(dev, seqlen),
                           SharedPrefix(pre, i64(dev, plen), i64(dev, of)), scale=0.125, once=once)
    for r, n in enumerate(seqlen):
        poison(own, r, n + 1, 70)
    for p, n in enumerate(plen[:2]):
        poison(pre, p, n, 200)
    poison(pre, 2, 0, 200)
    got = prefix_gqa_attn(bf16(dev, 4, 8, 1, 64, seed=20), own, i64(dev, seqlen),
                          SharedPrefix(pre, i64(dev, plen), i64(dev, of)), scale=0.125, once=once)
    assert torch.equal(got, want)


@pytest.mark.parametrize("once", [False, True])
def test_prefix_stays_with_its_rows(dev, once):
    """A NaN in a prefix reaches the rows that begin with it and no other."""
    from maple_amd.kernels import SharedPrefix, prefix_gqa_attn

    own, pre = make(dev, False, 40, 2, 20, 64, 72), make(dev, False, 2, 2, 100, 64, 74)
    poison(pre, 1, 3, 4)
    of = [i % 3 - 1 for i in range(40)]
    out = prefix_gqa_attn(bf16(dev, 40, 16, 1, 64), own, i64(dev, [19] * 40),
                          SharedPrefix(pre, i64(dev, [100, 100]), i64(dev, of)), scale=0.125, once=once)
    for r in range(40):
        assert (torch.isnan(out[r]).all() if of[r] == 1 else torch.isfinite(out[r]).all())


def test_prefix_same_as_a_joined_cache(dev):
    """The prefix copied into every row: the same output up to rounding of the weights, bf16 and quantised."""
    from maple_amd.kernels import KV, QuantKV, SharedPrefix, decode_gqa_attn, prefix_gqa_attn, quant_gqa_attn

    for quant, once in ((False, False), (False, True), (True, False), (True, True)):
        own, pre = make(dev, quant, 3, 2, 40, 64, 76), make(dev, quant, 1, 2, 128, 64, 78)
        both = [torch.cat([p.view(torch.uint8).expand(3, *p.view(torch.uint8).shape[1:]), o.view(torch.uint8)],
                          2).view(o.dtype) for p, o in zip(pre, own)]
        q, n = bf16(dev, 3, 8, 1, 64, seed=80), i64(dev, [39, 39, 39])
        a = prefix_gqa_attn(q, own, n, SharedPrefix(pre, i64(dev, [128]), i64(dev, [0, 0, 0])), scale=0.125, once=once)
        b = (quant_gqa_attn(q, QuantKV(*both), n + 128, scale=0.125) if quant else
             decode_gqa_attn(q, *both, n + 128, scale=0.125, window=None))
        k, v = values(QuantKV(*both) if quant else KV(*both))
        for r in range(3):
            _, mag = oq.attend(np64(q)[r, :, 0], k[r], v[r], 0.125)
            d = np.abs(np64(a)[r, :, 0] - np64(b)[r, :, 0])
            assert (d <= 2 * ((2.0 ** -8 + 2.0 ** -7 + 2.0 ** -12) * mag)).all()


# ---------------------------------------------------------------------------
# A step's token from its projection on
# ---------------------------------------------------------------------------
def check_fused(dev, seqlen, heads, rot=32, *, max_len=200, positions=None, norm=True, rows=None, row_map=None,
                table=torch.float32, w_dtype=torch.float32, qkv=None, window=None, scale=None, seed=0):
    """``quant_attention`` stores what ``apply_qkv_quant`` does, to the bit, and attends with its q."""
    from maple_amd.kernels import QuantKV, apply_qkv_quant, quant_attention

    nq, nkv, d = heads
    b = len(seqlen)
    qkv = bf16(dev, b, (nq + 2 * nkv) * d, seed=seed) if qkv is None else qkv
    cache = filled(dev, rows or b, nkv, max_len, d, seed=seed + 1)
    for r, n in enumerate(seqlen):  # what lies at the token's place and behind it does not matter
        poison(cache, r if row_map is None else row_map[r], min(max(n, 0), max_len), max_len)
    other = QuantKV(*(t.view(torch.uint8).clone().view(t.dtype) for t in cache))
    qw = kw = None
    if norm:
        qw, kw = ((torch.rand(d, device=dev) + 0.5).to(w_dtype) for _ in range(2))
    cos, sin = tables(max_len + 64, max(rot, 2), dev, table)
    scale = d ** -0.5 if scale is None else scale
    args = (qkv, qw, kw, cos, sin)
    more = dict(positions=i64(dev, positions), row_map=i64(dev, row_map), num_heads=nq, num_kv_heads=nkv, head_dim=d,
                rotary_dim=rot, use_rope=rot > 0, eps=EPS)
    out = quant_attention(*args, cache, i64(dev, seqlen), scale=scale, window=window, **more)
    q = apply_qkv_quant(*args, other, i64(dev, seqlen), **more)
    assert all(torch.equal(x, y) for x, y in zip(bits(cache), bits(other)))
    assert out.shape == q.shape and out.dtype == torch.bfloat16
    k, v = values(cache)
    for r in range(b):
        cr = r if row_map is None else row_map[r]
        ks, vs = oq.sequence((k[cr], v[cr]), min(seqlen[r] + 1, max_len), None, 0, window)
        within(np64(out)[r, :, 0], *oq.attend(np64(q)[r, :, 0], ks, vs, scale))


@pytest.mark.parametrize("heads", HEADS + [(16, 1, 128)])
@pytest.mark.parametrize("rot", [0, 20, 64])
def test_fused_layouts(dev, heads, rot):
    check_fused(dev, [0, 1, 31, 32, 33, 127, 128, 199], heads, rot)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 31, 64, 150, 2 ** 62])
def test_fused_windows(dev, d, window):
    check_fused(dev, [0, 1, 31, 63, 64, 65, 150, 199], (8, 2, d), window=window)


@pytest.mark.parametrize("heads,n", [((8, 1, 64), 5000), ((16, 4, 128), 3001), ((32, 4, 64), 2048)])
def test_fused_long_and_split(dev, heads, n):
    check_fused(dev, [n - 1, n // 2, 0, 1023, 1024], heads, max_len=n)


def test_fused_rows_positions_and_places(dev):
    check_fused(dev, [-1, 3, 200, 2 ** 40, -2 ** 40, 199], (4, 2, 64), 64)  # no token; behind the cache's end
    check_fused(dev, [-1, 1999, 2000], (16, 2, 128), 64, max_len=2000)
    check_fused(dev, [3, 9], (4, 2, 64), positions=[100, -7])
    check_fused(dev, [3, 9, 150], (4, 1, 128), 64, rows=5, row_map=[4, 0, 2])
    check_fused(dev, [3, 70], (4, 1, 128), 64, norm=False)
    check_fused(dev, [i % 70 for i in range(300)], (8, 1, 64), 64, max_len=70)


@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("w_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_fused_dtypes(dev, table, w_dtype):
    check_fused(dev, [7, 101], (8, 2, 128), 128, table=table, w_dtype=w_dtype)


def test_fused_odd_rows(dev):
    w = (4 + 2 * 2) * 64
    check_fused(dev, [1, 2, 130], (4, 2, 64), 64, qkv=bf16(dev, 3, w + 5, seed=12)[:, 5:])
    check_fused(dev, [1, 2, 130], (16, 1, 128), 64, qkv=bf16(dev, 3, 18 * 128 + 1, seed=12)[:, 1:])


def test_fused_not_finite_stays_in_its_row(dev):
    from maple_amd.kernels import quant_attention

    qkv = bf16(dev, 3, 8 * 64, seed=14)
    qkv[0, 4 * 64 + 3] = float("nan")  # row 0, K head 0: query heads 0 and 1
    qkv[1, 7 * 64 + 9] = float("inf")  # row 1, V head 1: dim 9 of query heads 2 and 3
    c = filled(dev, 3, 2, 300, 64)
    cos, sin = tables(300, 64, dev)
    w = torch.ones(64, device=dev)
    out = quant_attention(qkv, w, w, cos, sin, c, i64(dev, [200, 2, 77]), num_heads=4, num_kv_heads=2, head_dim=64,
                          rotary_dim=64, scale=0.125)[:, :, 0]
    odd = torch.isnan(out)
    assert odd[0, :2].all() and odd[1, 2:, 9].all()
    odd[0, :2], odd[1, 2:, 9] = False, False
    assert not odd.any() and torch.isfinite(out[2]).all()


# ---------------------------------------------------------------------------
# Calls
# ---------------------------------------------------------------------------
def one_step(dev, cache, prefix, seqlen, qkv, w, cos, sin):
    """A decode step's calls: the store, then attention over what was stored."""
    from maple_amd.kernels import apply_qkv_quant, prefix_gqa_attn, quant_gqa_attn

    at = seqlen + prefix.length[prefix.of.clamp(min=0)] * (prefix.of >= 0)
    q = apply_qkv_quant(qkv, w, w, cos, sin, cache, seqlen, positions=at, num_heads=8, num_kv_heads=2, head_dim=64,
                        rotary_dim=32)
    return quant_gqa_attn(q, cache, seqlen, scale=0.125), prefix_gqa_attn(q, cache, seqlen, prefix, scale=0.125, once=True)


def step_inputs(dev, seed=90):
    from maple_amd.kernels import SharedPrefix

    cos, sin = tables(1000, 32, dev)
    return (filled(dev, 5, 2, 300, 64, seed=seed),
            SharedPrefix(filled(dev, 2, 2, 600, 64, seed=seed + 2), i64(dev, [600, 333]), i64(dev, [0, 1, 1, -1, 0])),
            i64(dev, [0, 128, 255, 31, 298]), bf16(dev, 5, 12 * 64, seed=seed + 4),
            torch.rand(64, device=dev) + 0.5, cos, sin)


def test_step_of_calls_as_the_oracle(dev):
    cache, prefix, seqlen, qkv, w, cos, sin = step_inputs(dev)
    alone, behind = one_step(dev, cache, prefix, seqlen, qkv, w, cos, sin)
    x, c_np, s_np = np64(qkv).reshape(5, 12, 64), np64(cos), np64(sin)
    k, v = values(cache)
    sk, sv = values(prefix.cache)
    n, plen, of = seqlen.tolist(), prefix.length.tolist(), prefix.of.tolist()
    from maple_amd.kernels import apply_qkv_quant

    at = [a + (plen[o] if o >= 0 else 0) for a, o in zip(n, of)]
    q = apply_qkv_quant(qkv, w, w, cos, sin, cache, seqlen, positions=i64(dev, at), num_heads=8, num_kv_heads=2,
                        head_dim=64, rotary_dim=32)
    for r in range(5):
        for h in range(2):  # the stored token is this step's
            ref, mag = ot.head(x[r, 8 + h], np64(w), c_np[at[r]], s_np[at[r]], 32, False, 1e-6)
            got = k[r, h, n[r]]
            # bf16, then e4m3 (at least half the largest code's step in 2^14)
            step = np.maximum(2.0 ** -4 * np.abs(ref), 2.0 ** -10 * np.abs(ref).max() / 224)
            assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -16 * mag + 1.01 * step).all()
        ks, vs = oq.sequence((k[r], v[r]), n[r] + 1)
        within(np64(alone)[r, :, 0], *oq.attend(np64(q)[r, :, 0], ks, vs, 0.125))
        pre = (sk[of[r]], sv[of[r]]) if of[r] >= 0 else None
        ks, vs = oq.sequence((k[r], v[r]), n[r] + 1, pre, plen[of[r]] if of[r] >= 0 else 0)
        within(np64(behind)[r, :, 0], *oq.attend(np64(q)[r, :, 0], ks, vs, 0.125))


def test_calls_repeat_their_bits(dev):
    s = step_inputs(dev)
    a = one_step(dev, *s)
    for _ in range(3):
        b = one_step(dev, *s)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_on_another_stream(dev):
    s = step_inputs(dev)
    want = one_step(dev, *s)
    st = torch.cuda.Stream(dev)
    st.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(st):
        got = one_step(dev, *s)
    torch.cuda.current_stream(dev).wait_stream(st)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_two_streams_at_once(dev):
    """The same calls on two streams with no order between them, over one cache."""
    from maple_amd.kernels import prefix_gqa_attn, quant_gqa_attn

    cache, prefix, seqlen, _, _, _, _ = step_inputs(dev)
    qs = [bf16(dev, 5, 8, 1, 64, seed=97 + i) for i in range(2)]

    def calls(q):
        return [quant_gqa_attn(q, cache, seqlen, scale=0.125)] + [
            prefix_gqa_attn(q, cache, seqlen, prefix, scale=0.125, once=once) for once in (False, True)]

    want = [calls(q) for q in qs]
    streams = [torch.cuda.Stream(dev) for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(calls(qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(want[i], outs))


def test_two_captured_graphs(dev):
    """Two graphs of the same calls over different states, replayed in turn with eager work between."""
    states = [step_inputs(dev, seed=90), step_inputs(dev, seed=190)]
    graphs, outs = [], []
    for s in states:
        one_step(dev, *s)
    torch.cuda.synchronize()
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(one_step(dev, *s))
        graphs.append(g)
    for turn in range(4):
        for i in (turn % 2, 1 - turn % 2):
            states[i][3].copy_(bf16(dev, 5, 12 * 64, seed=1000 + 10 * turn + i))  # this step's qkv
            states[i][2].add_(1 if turn else 0).clamp_(max=299)
            graphs[i].replay()
            other = torch.randn(1 << 16, device=dev).sum()  # eager work on the same allocator
            torch.cuda.synchronize()
            want = one_step(dev, *states[i])
            assert torch.equal(want[0], outs[i][0]) and torch.equal(want[1], outs[i][1])
            assert torch.isfinite(other)


def test_fused_captured_on_another_stream(dev):
    """Two graphs of the fused step, replayed in turn on another stream, each against an eager step from the same cache."""
    from maple_amd.kernels import QuantKV, quant_attention

    states = [step_inputs(dev, seed=90), step_inputs(dev, seed=290)]

    def step(s, cache):
        _, _, seqlen, qkv, w, cos, sin = s
        return quant_attention(qkv, w, w, cos, sin, cache, seqlen, num_heads=8, num_kv_heads=2, head_dim=64, rotary_dim=32,
                               scale=0.125)

    def copy(cache):
        return QuantKV(*(t.view(torch.uint8).clone().view(t.dtype) for t in cache))

    for s in states:
        step(s, copy(s[0]))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(s, s[0]))
        graphs.append(g)
    st = torch.cuda.Stream(dev)
    for turn in range(4):
        for i in (turn % 2, 1 - turn % 2):
            states[i][3].copy_(bf16(dev, 5, 12 * 64, seed=2000 + 10 * turn + i))
            states[i][2].add_(1 if turn else 0).clamp_(max=299)
            fresh = copy(states[i][0])
            want = step(states[i], fresh)
            st.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(st):
                graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(want, outs[i])
            assert all(torch.equal(x, y) for x, y in zip(bits(fresh), bits(states[i][0])))


def test_empty_batches(dev):
    from maple_amd.kernels import (SharedPrefix, apply_qkv_quant, dequantize_kv, make_quant_kv, prefix_gqa_attn,
                                   quant_attention, quant_gqa_attn, quantize_kv)

    c = make_quant_kv(2, 2, 16, 64, dev)
    none = i64(dev, [])
    cos, sin = tables(16, 32, dev)
    q = apply_qkv_quant(bf16(dev, 0, 8 * 64), None, None, cos, sin, c, none, row_map=none, num_heads=4, num_kv_heads=2,
                        head_dim=64, rotary_dim=32)
    assert q.shape == (0, 4, 1, 64)
    assert quant_gqa_attn(q, c, none, row_map=none, scale=1.0).shape == q.shape
    assert quant_attention(bf16(dev, 0, 8 * 64), None, None, cos, sin, c, none, row_map=none, num_heads=4, num_kv_heads=2,
                           head_dim=64, rotary_dim=32, scale=1.0).shape == q.shape
    assert prefix_gqa_attn(q, c, none, SharedPrefix(c, i64(dev, [3, 4]), none), row_map=none, scale=1.0).shape == q.shape
    assert dequantize_kv(c, 4, row_map=none).k.shape == (0, 2, 4, 64)
    x = bf16(dev, 2, 2, 0, 64)
    before = bits(c)
    quantize_kv(x, x, c)
    assert all(torch.equal(a, b) for a, b in zip(before, bits(c)))


def test_no_prefixes_at_all(dev):
    """A prefix cache of no rows, or of no positions: the rows' own positions."""
    c = filled(dev, 2, 2, 100, 64, seed=95)
    from maple_amd.kernels import SharedPrefix, make_quant_kv, prefix_gqa_attn, quant_gqa_attn

    for shape in ((0, 2, 10, 64), (2, 2, 0, 64)):
        empty = make_quant_kv(*shape, dev)
        q, n = bf16(dev, 2, 8, 1, 64, seed=96), i64(dev, [99, 20])
        a = prefix_gqa_attn(q, c, n, SharedPrefix(empty, i64(dev, [0] * shape[0]), i64(dev, [0, -1])), scale=0.125)
        assert torch.equal(a, quant_gqa_attn(q, c, n, scale=0.125))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("once", [False, True])
def test_prefixes_may_be_rows_of_the_same_cache(dev, quant, once):
    """Rows that begin with what another row of their own cache holds, none of it copied."""
    from maple_amd.kernels import KV, QuantKV, SharedPrefix, prefix_gqa_attn

    c = make(dev, quant, 4, 2, 300, 64, 150)
    other = (QuantKV if quant else KV)(*(b.view(t.dtype) for b, t in zip(bits(c), c)))
    q, n, of = bf16(dev, 4, 8, 1, 64, seed=151), i64(dev, [299, 20, -1, 130]), i64(dev, [-1, 0, 0, 3])
    got, want = (prefix_gqa_attn(q, c, n, SharedPrefix(p, i64(dev, [300, 7, 0, 129]), of), scale=0.125, once=once)
                 for p in (c, other))
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(bits(c), bits(other)))


def test_index_tensors_of_32_bits(dev):
    """Write positions, lengths, places and maps in int32 and strided: as in int64."""
    from maple_amd.kernels import SharedPrefix, apply_qkv_quant, prefix_gqa_attn, quant_attention, quantize_kv

    cos, sin = tables(400, 32, dev)
    k, v, qkv = bf16(dev, 3, 2, 40, 64, seed=160), bf16(dev, 3, 2, 40, 64, seed=161), bf16(dev, 3, 8 * 64, seed=162)
    pre = filled(dev, 2, 2, 90, 64, seed=163)

    def calls(at):
        c = filled(dev, 5, 2, 60, 64, seed=164)
        rm, n = at([4, 0, 2]), at([39, 17, -1])
        kw = dict(positions=at([100, 20, 3]), row_map=rm, num_heads=4, num_kv_heads=2, head_dim=64, rotary_dim=32)
        quantize_kv(k, v, c, start=at([0, 3, 7]), lengths=at([40, 12, 0]), row_map=rm)
        q = apply_qkv_quant(qkv, None, None, cos, sin, c, n, **kw)
        outs = [q, quant_attention(qkv, None, None, cos, sin, c, n, scale=0.125, **kw)]
        outs += [prefix_gqa_attn(q, c, n, SharedPrefix(pre, at([90, 33]), at([1, 0, -1])), row_map=rm, scale=0.125, once=o)
                 for o in (False, True)]
        return outs + bits(c)

    want = calls(lambda x: i64(dev, x))
    for got in (calls(lambda x: i64(dev, x).int()), calls(lambda x: i64(dev, [x, x]).t()[:, 1])):
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("once", [False, True])
def test_a_graph_follows_its_prefixes(dev, once):
    """Prefixes, their lengths and their rows changed in place between replays."""
    from maple_amd.kernels import SharedPrefix, prefix_gqa_attn

    own, pre = filled(dev, 6, 2, 40, 64, seed=170), filled(dev, 3, 2, 500, 64, seed=172)
    q, n = bf16(dev, 6, 8, 1, 64, seed=174), i64(dev, [39, 3, -1, 0, 17, 38])
    prefix = SharedPrefix(pre, i64(dev, [500, 0, 1]), i64(dev, [0, 0, 1, 2, -1, 7]))

    def call():
        return prefix_gqa_attn(q, own, n, prefix, scale=0.125, once=once)

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for length, of in (([500, 0, 1], [0, 0, 1, 2, -1, 7]), ([1, 499, 33], [2] * 6), ([0, 0, 0], [0, 1, 2, 0, 1, 2]),
                       ([64, 65, 500], [1, 2, 0, 1, -1, 1]), ([500, 500, 500], [-1] * 6)):
        prefix.length.copy_(i64(dev, length))
        prefix.of.copy_(i64(dev, of))
        for _ in range(2):
            g.replay()
            other = torch.randn(1 << 16, device=dev).sum()  # eager work on the same allocator
            torch.cuda.synchronize()
            assert torch.equal(out, call()) and torch.isfinite(other)
        check_attn(dev, own, n.tolist(), 8, prefix=(pre, length, of), q=q)
