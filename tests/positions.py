"""Inputs on which every position of a sequence shows in an attention's output.

Positions have ids: prefix positions 0 .. P - 1, then a row's own P .. P + N - 1 (row
``b`` sees its prefix's first ones and its own first ones, the last ``window`` of both).

* Equal weights: q is 0 and V is 1 in one dim at the id of that dim, else 0.  All
  weights are 1, their sum is a whole number below 2^24 and the joins' factors are 1,
  all exact in float32, so an output is 1 / n (a float32 quotient, within 2^-20, rounded
  to bf16, 2^-8) where the id is one of the n that the row sees, else exactly 0.  A position that is
  left out gives 0, one that is taken twice 2 / n.
* Sharp keys: K is the id's bits as +1 and -1, q 128 times a target's bits.  The
  target's score passes every other one by 256, so the others' weights are below
  2^-368 and are 0, the target's is 1 and the output its V, exactly (the bf16 value
  that it is).  A K that meets another position's V, or a lost target, gives another
  row."""

from __future__ import annotations

import torch

BITS = 16


def seen(prefix_max, own_max, seqlen, plen=(), of=None, window=None, device="cpu"):
    """Which ids each row sees: bool ``[B, prefix_max + own_max]``."""
    out = torch.zeros(len(seqlen), prefix_max + own_max, dtype=torch.bool, device=device)
    for b, n in enumerate(seqlen):
        p = of[b] if of is not None else -1
        behind = min(plen[p], prefix_max) if 0 <= p < len(plen) else 0
        own = min(max(n + 1, 0), own_max)
        lo = 0 if window is None else max(0, behind + own - window)
        out[b, lo:behind] = True
        out[b, prefix_max + max(0, lo - behind):prefix_max + own] = True
    return out


def chunks(ids, nkv, d):
    """How many fillings of V it takes until every id has had a dim."""
    return -(-ids // (nkv * d))


def one_hot(chunk, ids, nkv, d, device):
    """V of all ids ``[nkv, ids, d]``: KV head ``h``'s dim ``i`` is id ``(chunk nkv + h) d + i``'s."""
    v = torch.zeros(nkv, chunks(ids, nkv, d) * nkv * d, d, device=device, dtype=torch.bfloat16)
    h, i = torch.arange(nkv, device=device).view(-1, 1), torch.arange(d, device=device)
    v[h, (chunk * nkv + h) * d + i, i] = 1.0
    return v[:, :ids]


def check_equal_weights(out, seen_ids, chunk, nkv):
    """``out [B, H, D]`` of the call with ``one_hot(chunk)``."""
    b, nq, d = out.shape
    n = seen_ids.sum(1, dtype=torch.float64).clamp(min=1.0)
    want = torch.zeros(b, (chunk + 1) * nkv * d, device=out.device, dtype=torch.float64)
    m = min(want.shape[1], seen_ids.shape[1])
    want[:, :m] = seen_ids[:, :m].double() / n.unsqueeze(1)
    want = want[:, chunk * nkv * d:].view(b, nkv, 1, d)
    off = ((out.double().view(b, nkv, nq // nkv, d) - want).abs() > (2.0 ** -8 + 2.0 ** -20) * want).nonzero()
    bad = [f"row {r} id {(chunk * nkv + h) * d + i}: {float(out[r, h * (nq // nkv) + g, i])}, of {int(n[r])}"
           for r, h, g, i in off[:4].tolist()]
    assert not bad, bad


def bits(ids, d, device):
    """K of all ids ``[ids, d]``: each id's lower bits as +1 and -1, then 0."""
    k = torch.zeros(ids, d, device=device, dtype=torch.bfloat16)
    at = torch.arange(ids, device=device).unsqueeze(1) >> torch.arange(BITS, device=device)
    k[:, :BITS] = ((at & 1) * 2 - 1).to(torch.bfloat16)
    return k


def targets(call, seen_ids, nq):
    """An id that the row sees for every row and query head, other ones each call: ``[B, H]`` (0 where there is none)."""
    n = seen_ids.sum(1)
    at = (call * nq + torch.arange(nq, device=seen_ids.device)) % n.clamp(min=1).unsqueeze(1)
    rank = seen_ids.cumsum(1) * seen_ids  # (1 at the first that is seen)
    return torch.searchsorted(torch.where(rank > 0, rank, 0).cummax(1).values, at + 1).clamp(max=seen_ids.shape[1] - 1)


def check_sharp(out, want, what=""):
    """``out`` against the targets' V, both ``[B, H, D]``."""
    off = (out.double() != want.double()).any(-1).nonzero()
    assert off.numel() == 0, f"{what}: other than the target's V at (row, head) {off[:8].tolist()} of {off.shape[0]}"
