"""The inputs of ``positions.py`` show a position that is lost, taken twice or paired
with another's V, and a window that is off by one: mistakes planted in the oracle."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import positions as pos
from oracle import quant_cache as oq

NKV, NQ, D = 2, 4, 64
P, N = 300, 200
SEQLEN, PLEN, OF = [199, 120, -1, 0, -1], [300, 77], [0, 1, 0, -1, -1]


def _oracle(q, k, v, seen_ids, edit=lambda ids: ids, shift=0):
    """Each row over the ids that it sees, in order; ``edit`` changes their list and ``shift`` moves V against K."""
    out = torch.zeros(*q.shape, dtype=torch.bfloat16)
    for b in range(q.shape[0]):
        ids = seen_ids[b].nonzero().flatten().tolist()
        ids = edit(ids) if ids else ids
        at = np.array(ids, dtype=np.int64)
        vs = v[:, np.roll(at, shift)]
        out[b] = torch.from_numpy(oq.attend(q[b], k[:, at], vs, 1.0)[0]).bfloat16()
    return out


def _equal(seen_ids, edit=lambda ids: ids, wrong=None):
    k = np.random.default_rng(1).normal(size=(NKV, P + N, D))
    for c in range(pos.chunks(P + N, NKV, D)):
        v = pos.one_hot(c, P + N, NKV, D, "cpu").double().numpy()
        out = _oracle(np.zeros((len(SEQLEN), NQ, D)), k, v, seen_ids if wrong is None else wrong, edit)
        pos.check_equal_weights(out, seen_ids, c, NKV)


@pytest.mark.parametrize("window", [None, 1, 130, 250, 10_000])
def test_equal_weights_as_the_oracle(window):
    _equal(pos.seen(P, N, SEQLEN, PLEN, OF, window))


@pytest.mark.parametrize("at", [0, 31, 32, 63, 77, 120, -32, -1])
@pytest.mark.parametrize("twice", [False, True])
def test_equal_weights_show_a_lost_or_doubled_position(at, twice):
    def edit(ids):
        at_ = at % len(ids)
        return ids[:at_] + ([ids[at_]] * 2 if twice else []) + ids[at_ + 1:]

    with pytest.raises(AssertionError):
        _equal(pos.seen(P, N, SEQLEN[:1], PLEN, OF[:1]).expand(len(SEQLEN), -1), edit)


@pytest.mark.parametrize("by", [-1, 1])
def test_equal_weights_show_a_window_off_by_one(by):
    with pytest.raises(AssertionError):
        _equal(pos.seen(P, N, SEQLEN, PLEN, OF, 130), wrong=pos.seen(P, N, SEQLEN, PLEN, OF, 130 + by))


def _sharp(seen_ids, edit=lambda ids: ids, shift=0):
    k = pos.bits(P + N, D, "cpu")
    v = torch.randn(NKV, P + N, D, generator=torch.Generator().manual_seed(2)).bfloat16()
    for call in range(-(-(P + N) // NQ)):
        t = pos.targets(call, seen_ids, NQ)
        q = (128.0 * k[t]).double().numpy()
        out = _oracle(q, k.double().expand(NKV, -1, -1).numpy(), v.double().numpy(), seen_ids, edit, shift)
        want = v[torch.arange(NQ) // (NQ // NKV), t] * seen_ids.any(1).view(-1, 1, 1)
        pos.check_sharp(out, want)


@pytest.mark.parametrize("window", [None, 130])
def test_sharp_keys_as_the_oracle(window):
    s = pos.seen(P, N, SEQLEN, PLEN, OF, window)
    _sharp(s)
    hit = torch.zeros_like(s)
    for call in range(-(-(P + N) // NQ)):
        hit.scatter_(1, pos.targets(call, s, NQ), True)
    assert torch.equal(hit & s, s) and not (hit & ~s)[s.any(1)].any()  # all that a row sees, and nothing else


@pytest.mark.parametrize("mistake", [dict(edit=lambda ids: ids[1:]), dict(edit=lambda ids: ids[:-1]), dict(shift=1),
                                     dict(edit=lambda ids: ids[:len(ids) // 2] + ids[len(ids) // 2 + 1:])],
                         ids=["first lost", "last lost", "V shifted", "middle lost"])
def test_sharp_keys_show_mistakes(mistake):
    with pytest.raises(AssertionError):
        _sharp(pos.seen(P, N, SEQLEN[:2], PLEN, OF[:2]), **mistake)
