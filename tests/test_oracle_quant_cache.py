"""The quantised cache's oracle (oracle/quant_cache.py) against its definitions."""

from __future__ import annotations

import numpy as np
import torch

from oracle import quant_cache as oq


def e4m3_values():
    v = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    return np.unique(v[np.isfinite(v)])


def test_codes_are_the_nearest_values_ties_to_even():
    v = e4m3_values()
    assert v.max() == oq.MOST
    assert (oq.e4m3(v) == v).all()
    lo, hi = v[:-1], v[1:]
    mid = (lo + hi) / 2
    near = oq.e4m3(mid)
    even = {x: i for i, x in enumerate(v[v >= 0])}  # a value's code, its last bit the mantissa's
    for m, a, b, r in zip(mid, lo, hi, near):
        assert r in (a, b)
        assert even[abs(r)] % 2 == 0, m
    eps = 1e-9
    assert (oq.e4m3(mid + eps * np.abs(mid) + 1e-15) == hi).all()
    assert (oq.e4m3(mid - eps * np.abs(mid) - 1e-15) == lo).all()
    assert oq.e4m3([1e9, -1e9]).tolist() == [448.0, -448.0]
    assert np.isnan(oq.e4m3([np.inf, -np.inf, np.nan])).all()


def test_codes_agree_with_torch_inside_the_range():
    x = np.random.default_rng(0).normal(size=20000) * 2.0 ** np.random.default_rng(1).integers(-12, 8, 20000)
    x = x[np.abs(x) <= 448]
    assert (oq.e4m3(x) == torch.tensor(x).to(torch.float8_e4m3fn).double().numpy()).all()


def test_scale_is_the_least_power():
    rng = np.random.default_rng(2)
    rows = [rng.normal(size=8) * 2.0 ** s for s in range(-120, 121, 7)]
    rows += [np.full(8, 448.0 * 2.0 ** s) for s in (-126, -3, 0, 5, 119)]
    rows += [np.full(8, np.nextafter(448.0, 500.0) * 2.0 ** s) for s in (-126, -3, 0, 5, 118)]
    e = oq.exponent(np.stack(rows))
    for row, got in zip(rows, e):
        fits = [p for p in range(oq.LOW, oq.HIGH + 1) if np.abs(row).max() <= 448.0 * 2.0 ** p]
        assert got == (min(fits) if fits else oq.HIGH)
    assert oq.exponent(np.zeros((1, 4)))[0] == oq.LOW
    assert oq.exponent(np.array([[1.0, np.inf, np.nan]]))[0] == oq.exponent(np.array([[1.0]]))[0]
    assert oq.exponent(np.array([[3.3e38]]))[0] == oq.HIGH


def test_decoded_values_are_within_half_a_step():
    x = np.random.default_rng(3).normal(size=(50, 64))
    c, e = oq.encode(x)
    y = oq.decode(c, e)
    assert (np.abs(y - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** (e[:, None] - 10.0))).all()


def test_attention_by_hand_and_joined():
    rng = np.random.default_rng(4)
    q, k, v = rng.normal(size=(4, 8)), rng.normal(size=(2, 9, 8)), rng.normal(size=(2, 9, 8))
    one, _ = oq.attend(q, k[:, :1], v[:, :1], 0.3)
    assert np.allclose(one, np.repeat(v[:, 0], 2, 0))
    same, _ = oq.attend(np.zeros_like(q), k, v, 0.3)
    assert np.allclose(same, np.repeat(v.mean(1), 2, 0))
    assert (oq.attend(q, k[:, :0], v[:, :0], 0.3)[0] == 0).all()
    pk, pv = oq.sequence((k[:, 5:], v[:, 5:]), 4, (k[:, :5], v[:, :5]), 5)
    assert (pk == k).all() and (pv == v).all()
    wk, _ = oq.sequence((k[:, 5:], v[:, 5:]), 4, (k[:, :5], v[:, :5]), 5, window=6)
    assert (wk == k[:, 3:]).all()
    none, _ = oq.sequence((k, v), 0, (k[:, :5], v[:, :5]), 2)
    assert (none == k[:, :2]).all()
