"""A quantised KV cache and attention over it and over shared prefixes, NumPy in
float64 (test infrastructure only: the product never imports it).

Restates ``maple_amd/kernels/quant_cache.py`` from its definitions; no reference
counterpart.  Pinned in ``tests/test_oracle_quant_cache.py``: the codes against
every e4m3 value and the midpoints between neighbours, the scale against its
definition by trying all powers, attention with a prefix against attention over
the joined sequence written out, and one key's by hand.
"""

from __future__ import annotations

import numpy as np

MOST = 448.0
LOW, HIGH = -126, 119


def e4m3(x):
    """The e4m3 value nearest (even) to each finite ``x``, at most 448 in size; NaN for others."""
    x = np.asarray(x, np.float64)
    out = np.full(x.shape, np.nan)
    ok = np.isfinite(x)
    a = np.abs(x[ok])
    e = np.maximum(np.frexp(np.maximum(a, 2.0 ** -30))[1] - 1, -6)  # exponent of the binade, least normal 2^-6
    step = 2.0 ** (e - 3.0)
    out[ok] = np.copysign(np.minimum(np.rint(a / step) * step, MOST), x[ok])
    return out


def exponent(x):
    """Per row (last axis) the least e with max |finite x| <= 448 * 2^e, in [-126, 119]."""
    x = np.asarray(x, np.float64)
    top = np.where(np.isfinite(x), np.abs(x), 0.0).max(-1)
    m, p = np.frexp(top)  # top = m 2^p, m in [1/2, 1); 448 = (7/8) 2^9
    e = np.where(m <= 0.875, p - 9, p - 8)
    return np.clip(np.where(top == 0, LOW, e), LOW, HIGH)


def encode(x):
    """``(codes as their values, exponents)`` of rows."""
    e = exponent(x)
    with np.errstate(invalid="ignore", over="ignore"):
        return e4m3(np.asarray(x, np.float64) * 2.0 ** -e[..., None].astype(np.float64)), e


def decode(codes, e):
    return np.asarray(codes, np.float64) * 2.0 ** np.asarray(e, np.float64)[..., None]


def attend(q, k, v, scale: float):
    """One row: ``q [H, D]`` over ``k`` / ``v [Hkv, n, D]``; returns the output ``[H, D]`` and
    ``sum p |v|`` (what its rounding scales with); 0 where ``n`` is 0."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    h, d = q.shape
    n_kv, n, _ = k.shape
    if n == 0:
        return np.zeros((h, d)), np.zeros((h, d))
    g = h // n_kv
    x = np.einsum("hgd,hnd->hgn", q.reshape(n_kv, g, d), k) * scale
    p = np.exp(x - x.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return np.einsum("hgn,hnd->hgd", p, v).reshape(h, d), np.einsum("hgn,hnd->hgd", p, np.abs(v)).reshape(h, d)


def sequence(own, n_own: int, prefix=None, n_prefix: int = 0, window=None):
    """A row's ``(k, v) [Hkv, n, D]``: the prefix's first positions, its own, the last ``window`` of both."""
    k, v = own[0][:, :max(n_own, 0)], own[1][:, :max(n_own, 0)]
    if prefix is not None:
        k, v = (np.concatenate([p[:, :n_prefix], t], 1) for p, t in zip(prefix, (k, v)))
    if window is not None:
        n = k.shape[1]
        k, v = k[:, max(0, n - window):], v[:, max(0, n - window):]
    return k, v
