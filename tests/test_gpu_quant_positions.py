"""Every position that a row sees counts once in the attention over quantised caches
and shared prefixes, and no other counts: outputs by the inputs of ``positions.py``, whose
docstring derives the bounds, over sequences whose splits, rounds of tiles, tiles and
joins all end somewhere among the tested positions.

Splits of a row, by the plan: 2 rows of 4 KV heads over 5003 positions 32 (20 of them
with positions), 16 rows 8 of five rounds of 128 each; 2 rows over 3001 24; one row over
20000 157, over 4097 33; under windows of 1000 and 1025 4 to 9, of 3000 4 to 24.  Behind
the prefixes of up to 2050 21 where each row reads them, 17 of a prefix where it is read
once; behind the one of 4801 52, and 40 beside 12 of the rows' own positions."""

from __future__ import annotations

import pytest
import torch

import positions as pos

pytestmark = pytest.mark.gpu


def i64(dev, x):
    return torch.tensor(x, device=dev, dtype=torch.int64)


def cache_of(k, v, quant):
    """A cache of bf16 ``k`` and ``v``; ±1, 0 and 1 are codes."""
    from maple_amd.kernels import KV, make_quant_kv, quantize_kv

    return quantize_kv(k, v, make_quant_kv(*k.shape, k.device)) if quant else KV(k.contiguous(), v.contiguous())


def code_values(v):
    """bf16 values as a quantised cache holds them."""
    from maple_amd.kernels import dequantize_kv, make_quant_kv, quantize_kv

    return dequantize_kv(quantize_kv(v, v, make_quant_kv(*v.shape, v.device))).k


class Case:
    """A call over sequences of ``n`` own positions behind prefixes of ``p`` (0: none), by ``form``:
    own (``quant_gqa_attn``), fused (``quant_attention``), or once / each / default of ``prefix_gqa_attn``."""

    def __init__(self, dev, heads, n, seqlen, *, form="own", window=None, p=0, plen=(), of=None, quant=True):
        self.dev, self.n, self.p, self.form, self.window, self.quant = dev, n, p, form, window, quant
        self.nq, self.nkv, self.d = heads
        self.seqlen, self.plen, self.of = seqlen, plen, of
        self.seen = pos.seen(p, n, seqlen, plen, of, window, dev)

    def spread(self, x, rows, lo, hi):
        """Ids ``lo .. hi`` of ``x [nkv, ids, D]`` in each of ``rows`` cache rows."""
        return x[:, lo:hi].unsqueeze(0).expand(rows, -1, -1, -1)

    def run(self, q, k, v):
        """``q [B, H, D]``, K and V of all ids ``[nkv, ids, D]``."""
        from maple_amd.kernels import SharedPrefix, prefix_gqa_attn, quant_attention, quant_gqa_attn

        b, n, p = len(self.seqlen), self.n, self.p
        sl, kw = i64(self.dev, self.seqlen), dict(scale=1.0, window=self.window)
        if self.form == "fused":
            own_k, own_v = self.spread(k, b, p, p + n).clone(), self.spread(v, b, p, p + n).clone()
            at = sl.clamp(0, n - 1)
            r = torch.arange(b, device=self.dev)
            new = torch.cat([q, own_k[r, :, at], own_v[r, :, at]], 1).view(b, -1)
            there = ((sl >= 0) & (sl < n)).nonzero().flatten()
            own_k[there, :, at[there]] = 3.0  # (the token's place: what lies there does not matter)
            own_v[there, :, at[there]] = 5.0
            return quant_attention(new, None, None, None, None, cache_of(own_k, own_v, True), sl, num_heads=self.nq,
                                   num_kv_heads=self.nkv, head_dim=self.d, rotary_dim=0, use_rope=False, **kw)[:, :, 0]
        own = cache_of(self.spread(k, b, p, p + n), self.spread(v, b, p, p + n), self.quant)
        q = q.unsqueeze(2)
        if self.form == "own":
            return quant_gqa_attn(q, own, sl, **kw)[:, :, 0]
        pre = cache_of(self.spread(k, len(self.plen), 0, p), self.spread(v, len(self.plen), 0, p), self.quant)
        once = {"once": True, "each": False, "default": None}[self.form]
        return prefix_gqa_attn(q, own, sl, SharedPrefix(pre, i64(self.dev, self.plen), i64(self.dev, self.of)), once=once,
                               **kw)[:, :, 0]

    def equal_weights(self):
        ids = self.p + self.n
        q = torch.zeros(len(self.seqlen), self.nq, self.d, device=self.dev, dtype=torch.bfloat16)
        k = torch.randn(self.nkv, ids, self.d, generator=torch.Generator(self.dev).manual_seed(1), device=self.dev).bfloat16()
        for c in range(pos.chunks(ids, self.nkv, self.d)):
            pos.check_equal_weights(self.run(q, k, pos.one_hot(c, ids, self.nkv, self.d, self.dev)), self.seen, c, self.nkv)

    def sharp(self):
        """Each seen position in turn the target."""
        ids = self.p + self.n
        k = pos.bits(ids, self.d, self.dev)
        v = torch.randn(1, self.nkv, ids, self.d, generator=torch.Generator(self.dev).manual_seed(2), device=self.dev).bfloat16()
        held = (code_values(v) if self.quant else v)[0]
        most = -(-int(self.seen.sum(1).max()) // self.nq)
        head = torch.arange(self.nq, device=self.dev) // (self.nq // self.nkv)
        for call in range(most):
            t = pos.targets(call, self.seen, self.nq)
            out = self.run(128.0 * k[t], k.expand(self.nkv, -1, -1), held)
            pos.check_sharp(out, held[head, t] * self.seen.any(1).view(-1, 1, 1), f"call {call}")


TWO = [5002, 4864]
MANY = [5002, 5001, 4095, 4096, 4097, 1279, 1280, 1281, 639, 640, 127, 128, 0, -1, 2 ** 40, 2559]
OWN = {
    "2 x 5003": ((8, 4, 64), 5003, TWO),
    "16 x 5003": ((8, 4, 64), 5003, MANY),
    "2 x 3001 of 128": ((16, 4, 128), 3001, [3000, 1500]),
    "1 x 20000": ((8, 1, 64), 20000, [19999]),
    "1 x 4097 of 128": ((3, 1, 128), 4097, [4096]),
}
OWN_CASES = pytest.mark.parametrize("case", OWN, ids=list(OWN))
FORMS = pytest.mark.parametrize("form", ["own", "fused"])


@FORMS
@OWN_CASES
def test_every_position_counts_once(dev, case, form):
    Case(dev, *OWN[case], form=form).equal_weights()


@FORMS
@pytest.mark.parametrize("case", ["2 x 5003", "16 x 5003", "2 x 3001 of 128", "1 x 4097 of 128"])
@pytest.mark.parametrize("window", [1000, 1025, 3000])
def test_a_window_over_splits(dev, case, window, form):
    """Windows that begin inside a row and are split, rows shorter than them among the rest."""
    Case(dev, *OWN[case], form=form, window=window).equal_weights()


@FORMS
@pytest.mark.parametrize("case,window", [("2 x 5003", None), ("16 x 5003", None), ("16 x 5003", 1025),
                                         ("2 x 3001 of 128", None), ("2 x 3001 of 128", 1000), ("1 x 4097 of 128", None)])
def test_each_key_meets_its_value(dev, case, window, form):
    Case(dev, *OWN[case], form=form, window=window).sharp()


BEHIND = {
    "two of 2050": dict(heads=(8, 2, 64), n=700, seqlen=[699, 300, -1, 650, 0, 127], p=2050, plen=[2050, 1025],
                        of=[0, 1, 0, -1, 1, 0]),
    "one of 4801, 128": dict(heads=(16, 1, 128), n=1500, seqlen=[1499, 700, -1], p=5000, plen=[4801], of=[0, 0, 0]),
}
PREFIX_CASES = pytest.mark.parametrize("case", BEHIND, ids=list(BEHIND))
KINDS = pytest.mark.parametrize("quant", [False, True], ids=["bf16", "quantised"])


@KINDS
@pytest.mark.parametrize("form", ["once", "each", "default"])
@PREFIX_CASES
def test_every_position_behind_a_prefix_counts_once(dev, case, form, quant):
    Case(dev, **BEHIND[case], form=form, quant=quant).equal_weights()


@KINDS
@pytest.mark.parametrize("window", [1000, 1025, 3000])
@PREFIX_CASES
def test_a_window_that_begins_in_a_prefix(dev, case, window, quant):
    Case(dev, **BEHIND[case], form="each", window=window, quant=quant).equal_weights()


@KINDS
@pytest.mark.parametrize("form", ["once", "each"])
@PREFIX_CASES
def test_each_key_behind_a_prefix_meets_its_value(dev, case, form, quant):
    Case(dev, **BEHIND[case], form=form, quant=quant).sharp()


@KINDS
@PREFIX_CASES
def test_each_key_in_a_window_meets_its_value(dev, case, quant):
    Case(dev, **BEHIND[case], form="each", window=1025, quant=quant).sharp()


def _random(case):
    """Random q, K and V for a case, one draw."""
    g = torch.Generator(case.dev).manual_seed(7)

    def draw(*shape):
        return torch.randn(shape, generator=g, device=case.dev).bfloat16()

    ids = case.p + case.n
    return draw(len(case.seqlen), case.nq, case.d), draw(case.nkv, ids, case.d), draw(case.nkv, ids, case.d)


@FORMS
@OWN_CASES
def test_split_calls_repeat_their_bits(dev, case, form):
    c = Case(dev, *OWN[case], form=form)
    q, k, v = _random(c)
    q = q * c.d ** -0.5
    first = c.run(q, k, v)
    assert all(torch.equal(first, c.run(q, k, v)) for _ in range(5))


@KINDS
@pytest.mark.parametrize("form", ["once", "each"])
@PREFIX_CASES
def test_split_calls_behind_a_prefix_repeat_their_bits(dev, case, form, quant):
    c = Case(dev, **BEHIND[case], form=form, quant=quant)
    q, k, v = _random(c)
    q = q * c.d ** -0.5
    first = c.run(q, k, v)
    assert all(torch.equal(first, c.run(q, k, v)) for _ in range(5))
