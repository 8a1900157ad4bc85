"""Rotary tables scaled for long contexts (model.RopeScaling, CPU): the
published definitions, term by term in 64 bits, and the table built without
scaling as it was."""

from __future__ import annotations

import math

import pytest
import torch

from maple_amd.model import DecoderConfig, RopeScaling, rope_tables

# float32 tables of values up to 1.3: one rounding
ATOL = 2.0 ** -23


def _check(scaling, rot, freq, mult=1.0, theta=10000.0):
    n = 70001
    cos, sin = rope_tables(n, rot, theta, "cpu", scaling)
    assert cos.shape == sin.shape == (n, rot) and cos.dtype == sin.dtype == torch.float32
    for pos in (0, 1, 4095, 70000):
        for i in range(rot // 2):
            a = pos * freq(i)
            for col in (i, i + rot // 2):
                # (pos * freq rounds once in 64 bits, 2^-53 of up to 7e4)
                assert abs(cos[pos, col].item() - mult * math.cos(a)) <= ATOL
                assert abs(sin[pos, col].item() - mult * math.sin(a)) <= ATOL


def test_linear_divides_positions():
    _check(RopeScaling("linear", 8.0), 32, lambda i: 10000.0 ** (-2 * i / 32) / 8.0)


def test_ntk_keeps_the_fastest_and_divides_the_slowest():
    base = 10000.0 * 4.0 ** (64 / 62)
    _check(RopeScaling("ntk", 4.0), 64, lambda i: base ** (-2 * i / 64))
    inv, _ = RopeScaling("ntk", 4.0).frequencies(64, 10000.0, "cpu")
    plain = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert inv[0] == 1.0 and abs(inv[-1].item() * 4.0 / plain[-1].item() - 1.0) < 1e-12


def test_yarn_blends_by_turns():
    s = RopeScaling("yarn", 16.0, original_len=4096)

    def freq(i):
        f = 10000.0 ** (-2 * i / 128)
        turns = 4096 * f / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / 31.0))
        return keep * f + (1 - keep) * f / 16.0

    _check(s, 128, freq, 0.1 * math.log(16.0) + 1.0)


def test_factor_one_changes_nothing_but_rounding():
    plain = rope_tables(64, 32, 10000.0, "cpu")
    for kind in ("linear", "ntk", "yarn"):
        for a, b in zip(plain, rope_tables(64, 32, 10000.0, "cpu", RopeScaling(kind, 1.0))):
            # (the plain table's angles are float32: 64 * 2^-23, twice)
            assert (a - b).abs().max() <= 2 * 64 * 2.0 ** -23


@pytest.mark.parametrize("bad", [dict(kind="x", factor=2.0), dict(kind="linear", factor=0.5),
                                 dict(kind="ntk", factor=float("inf")), dict(kind="yarn", factor=2.0, original_len=0),
                                 dict(kind="yarn", factor=2.0, slow=40.0)])
def test_refusals(bad):
    with pytest.raises(ValueError):
        RopeScaling(**bad)


def test_ntk_needs_two_frequencies_and_configs_default_to_none():
    with pytest.raises(ValueError):
        rope_tables(4, 2, 10000.0, "cpu", RopeScaling("ntk", 2.0))
    assert DecoderConfig().rope_scaling is None


def test_checkpoints_keep_the_scaling(tmp_path):
    from maple_amd import checkpoint
    from maple_amd.model import SyntheticDecoder

    cfg = DecoderConfig(hidden=256, layers=1, heads=4, kv_heads=2, head_dim=64, experts=8, inter=256, top_k=2,
                        vocab=256, rope_scaling=RopeScaling("yarn", 4.0, original_len=32))
    model = SyntheticDecoder(cfg, "cpu", seed=1, max_len=128)
    checkpoint.save_decoder(model, tmp_path)
    back = checkpoint.load_decoder(tmp_path, "cpu", max_len=128)
    assert back.cfg.rope_scaling == cfg.rope_scaling
    assert torch.equal(back.cos, model.cos) and torch.equal(back.sin, model.sin)
    want = rope_tables(128, 32, 10000.0, "cpu", cfg.rope_scaling)
    assert torch.equal(model.cos, want[0]) and torch.equal(model.sin, want[1])
