"""Decoding with trees of drafted tokens, NumPy in float64 (test infrastructure
only: the product never imports it).

Restates ``maple_amd/kernels/tree.py`` node by node from its definitions; no
reference counterpart.  Pinned in ``tests/test_oracle_tree.py``: ancestors by
hand and against walking up; a tree of one node against ``oracle.decoder`` and
``oracle.sampler``; a chain against causal attention row by row; the
verification against its purpose (summed over the draft's choices and a grid of
uniforms, the first emitted token follows the target's law) and against greedy
decoding.
"""

from __future__ import annotations

import numpy as np

from . import kernels as ok
from .sampler import topk_desc


def branches(parents) -> list:
    """Per node the nodes from the root down to it; None for an absent node."""
    p = [int(v) for v in parents]
    line = [[0] if p[0] == -1 else None]
    for i in range(1, len(p)):
        up = line[p[i]] if 0 <= p[i] < i else None
        line.append(None if up is None else up + [i])
    return line


def rotate(y, cos_row, sin_row, rot: int, interleaved: bool):
    """Rotary positions on the first ``rot`` dims of one head; returns the result
    and the sum of its two terms' magnitudes (what its float32 error scales
    with)."""
    y = np.asarray(y, np.float64)
    out, mag, h = y.copy(), np.abs(y), rot // 2
    for i in range(h):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
        out[a] = y[a] * cos_row[i] - y[b] * sin_row[i]
        out[b] = y[b] * cos_row[i + h] + y[a] * sin_row[i + h]
        mag[a] = abs(y[a] * cos_row[i]) + abs(y[b] * sin_row[i])
        mag[b] = abs(y[b] * cos_row[i + h]) + abs(y[a] * sin_row[i + h])
    return out, mag


def head(x, w, cos_row, sin_row, rot: int, interleaved: bool, eps: float):
    """RMSNorm (``w`` None: none) and rotary positions of one head."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt(np.mean(x * x) + eps) * np.asarray(w, np.float64)
    if not rot:
        return x, np.abs(x)
    return rotate(x, ok.bf16_round(cos_row).astype(np.float64), ok.bf16_round(sin_row).astype(np.float64), rot,
                  interleaved)


def seen(parents, seqlen: int, max_len: int, window=None) -> list:
    """Per node the cache positions that it attends; None for an absent node."""
    out = []
    for up in branches(parents):
        if up is None:
            out.append(None)
            continue
        at = seqlen + len(up) - 1  # the node's position
        lo = max(0, at + 1 - window) if window else 0
        near = up[-window:] if window else up
        out.append(list(range(lo, seqlen)) + [seqlen + a for a in near if seqlen + a < max_len])
    return out


def attention(q, k, v, positions, scale: float):
    """One node's heads ``q [H, D]`` over ``positions`` of ``k`` / ``v [Hkv, L, D]``;
    returns the output and ``sum p |v|`` (what the rounding of p scales with)."""
    nq, d = q.shape
    nkv = k.shape[0]
    out, mag = np.zeros((nq, d)), np.zeros((nq, d))
    if not positions:
        return out, mag
    kk, vv = np.asarray(k, np.float64)[:, positions], np.asarray(v, np.float64)[:, positions]
    for h in range(nq):
        s = kk[h * nkv // nq] @ np.asarray(q[h], np.float64) * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], mag[h] = p @ vv[h * nkv // nq], p @ np.abs(vv[h * nkv // nq])
    return out, mag


def law(logits, *, temperature: float, top_p: float, top_k: int):
    """The sampler's law at a node: ids (most likely first) and probabilities."""
    z = np.asarray(logits, np.float64)
    ids = topk_desc(z, top_k)
    low = np.zeros(ids.size)  # (equal logits weigh alike, infinite ones too)
    np.subtract(z[ids], z[ids[0]], out=low, where=z[ids] != z[ids[0]])
    p = np.exp(low / temperature)
    p /= p.sum()
    before = np.concatenate([[0.0], np.cumsum(p)[:-1]])
    p = np.where((before <= top_p) | (top_p >= 1.0), p, 0.0)
    return ids, p / p.sum()


def verify(logits, tokens, parents, uniform, *, temperature: float, top_p: float, top_k: int, probs=None):
    """One row: ``(emitted tokens, path)``; both empty for a row without a
    sequence.  ``logits [T, V]``, ``probs [T, V]`` or None."""
    line = branches(parents)
    if line[0] is None:
        return [], []
    kw = dict(temperature=temperature, top_p=top_p, top_k=top_k)
    cur, path, out = 0, [0], []
    ids, p = law(logits[0], **kw)
    while True:
        for c in range(cur + 1, len(parents)):
            if line[c] is None or int(parents[c]) != cur:
                continue
            t, u = int(tokens[c]), float(uniform[c])
            at = np.nonzero(ids == t)[0]
            pt = p[at[0]] if at.size else 0.0
            if probs is None:
                qt, q = 1.0, (ids == t).astype(np.float64)
            else:
                row = np.asarray(probs[c], np.float64)
                qt, q = (row[t] if 0 <= t < row.shape[0] else 0.0), row[ids]
            if u * qt < pt:
                out.append(t)
                path.append(c)
                cur = c
                ids, p = law(logits[c], **kw)
                break
            rest = np.maximum(p - q, 0.0)
            if rest.sum() > 0:
                p = rest / rest.sum()
        else:
            break
    cum = np.cumsum(p)
    out.append(int(ids[min(int((cum <= float(uniform[0]) * cum[-1]).sum()), top_k - 1)]))
    return out, path
