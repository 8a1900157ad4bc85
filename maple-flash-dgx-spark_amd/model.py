"""Synthetic packed decoder on the HIP kernels (decode path of reference
``src/maple_run/model.py``: ``MapleDecoderLayer`` :477-506,
``MapleForCausalLM.forward`` :848-886, ``KVCache`` :116-310).

One decode step, per layer:
  qkv   = ternary_gemv(hidden, W_qkv, rms_weight=input_ln)     (fused RMSNorm)
  attn  = decode_attention(qkv, ...)    QK-norm + RoPE, K/V written at seqlen,
                                        GQA over the cache (one launch)
  o     = ternary_gemv(attn, W_o)
  hidden, mlp_in = add_rms_norm(hidden, o, post_ln)
  hidden = moe_block(mlp_in, residual=hidden)
  (at batch 1, when the one-launch MoE kernel is built for the shape and
  fused_moe is left True, the last two lines are one launch:
  moe_fused(hidden, add=o, norm_weight=post_ln), which in forward() also
  computes the next layer's qkv line from its output, so only layer 0 runs
  the standalone QKV projection; from 17 tokens, with combine_next left True,
  the grouped MoE's top-k combine is left to the next layer's QKV projection,
  which builds hidden from the slot outputs in its operand launch)
then seqlen += 1, final rms_norm, RTN4 lm_head, greedy argmax.

A step over a tree of drafted tokens per row (``forward_tree``) runs the same
layers over all nodes at once, with ``apply_qkv_tree`` and ``tree_attention`` in
the place of ``decode_attention``; ``KVCache.commit`` then keeps an accepted
branch.

Over a quantised cache (``make_cache(quantized=True)``, ``KVCache.quantized``) the
attention of a step is ``quant_attention``, and over rows behind shared prefixes
(``KVCache.share``) the store and ``prefix_gqa_attn``, in the place of
``decode_attention``.

Weights are random with the synthetic distributions (``synthetic.py``): every
projection packed ternary, norm weights 1, the lm_head and embedding 4-bit RTN
with group 128 and zero-centred dequantised values, RoPE on every layer over
half the head (rotary_dim 32, theta 1e4), full attention (no window).
"""

from __future__ import annotations

import dataclasses
import math
from dataclasses import dataclass, field

import torch

from . import synthetic
from .kernels.decode_attn import apply_qkv_decode, decode_attention, gqa_workspace, o_projection_supported
from .kernels.fused_norm import rms_norm
from .kernels.greedy import greedy_argmax
from .kernels.quant_cache import (KV, QuantKV, SharedPrefix, apply_qkv_quant, dequantize_kv, make_quant_kv,
                                  prefix_gqa_attn, quant_attention, quantize_kv)
from .kernels.rtn4 import rtn4_embedding, rtn4_gemv
from .kernels.ternary_gemv import combine_gemv_supported, ternary_gemv, ternary_gemv_combine
from .kernels.tree import apply_qkv_tree, check_tree, commit_tree, tree_attention
from .moe import PendingCombine, fused_form, fused_supported, moe_fused, moe_layer


@dataclass(frozen=True)
class RopeScaling:
    """Rotary positions past the trained context, by a ``factor`` over
    ``original_len`` positions (published methods, angles in 64 bits):

    * ``"linear"``: positions divided by ``factor``;
    * ``"ntk"``: the base raised to ``theta * factor^(rot / (rot - 2))``, so that
      the slowest frequency is divided by ``factor`` and the fastest kept;
    * ``"yarn"``: a frequency that turns fewer than ``slow`` times in
      ``original_len`` positions is divided by ``factor``, one that turns more than
      ``fast`` times kept, those between blended linearly; cos and sin are multiplied by
      ``0.1 ln(factor) + 1``."""

    kind: str
    factor: float
    original_len: int = 4096
    slow: float = 1.0
    fast: float = 32.0

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "yarn"):
            raise ValueError(f"rope scaling {self.kind!r}: linear, ntk or yarn")
        if not (self.factor >= 1.0 and math.isfinite(self.factor)) or self.original_len < 1 or not (
                0.0 < self.slow < self.fast):
            raise ValueError(f"rope scaling needs factor >= 1, original_len >= 1 and 0 < slow < fast: {self}")

    def frequencies(self, rotary_dim: int, theta: float, device) -> tuple:
        """``(inv_freq [rotary_dim / 2] float64, factor of cos and sin)``."""
        i = torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64)
        if self.kind == "ntk":
            if rotary_dim <= 2:
                raise ValueError("ntk scaling needs a rotary_dim above 2")
            theta = theta * self.factor ** (rotary_dim / (rotary_dim - 2))
        inv = theta ** (-i / rotary_dim)
        if self.kind == "ntk":
            return inv, 1.0
        if self.kind == "linear":
            return inv / self.factor, 1.0
        turns = self.original_len * inv / (2.0 * math.pi)
        keep = ((turns - self.slow) / (self.fast - self.slow)).clamp(0.0, 1.0)
        return inv * keep + inv / self.factor * (1.0 - keep), 0.1 * math.log(self.factor) + 1.0


@dataclass
class DecoderConfig:
    hidden: int = 2048
    layers: int = 24
    heads: int = 32
    kv_heads: int = 4
    head_dim: int = 64
    experts: int = 64
    inter: int = 768
    top_k: int = 8
    vocab: int = 151936
    rtn_group: int = 128
    rope_theta: float = 10000.0
    partial_rotary: float = 0.5
    eps: float = 1e-6
    lm_scale: tuple = (0.003, 0.006)
    # per-layer attention (model.py:646-649, 784-786): "full_attention" or
    # "sliding_attention" (the last sliding_window positions); empty = all full.
    # nope_on_global: full-attention layers skip RoPE.
    layer_types: tuple = ()
    sliding_window: int = 512
    nope_on_global: bool = False
    rope_scaling: RopeScaling | None = None

    def layer_attention(self, i: int) -> tuple:
        """``(window or None, use_rope)`` of layer ``i``."""
        kind = self.layer_types[i] if self.layer_types else "full_attention"
        window = self.sliding_window if kind == "sliding_attention" else None
        return window, not (self.nope_on_global and kind == "full_attention")

    @property
    def qkv_rows(self) -> int:
        return (self.heads + 2 * self.kv_heads) * self.head_dim

    @property
    def rotary_dim(self) -> int:
        return int(self.head_dim * self.partial_rotary)


@dataclass
class DecoderLayerWeights:
    qkv: torch.Tensor
    qkv_alpha: torch.Tensor
    o: torch.Tensor
    o_alpha: torch.Tensor
    input_ln: torch.Tensor
    post_ln: torch.Tensor
    q_norm: torch.Tensor
    k_norm: torch.Tensor
    moe: synthetic.MoELayer


def rope_tables(max_len: int, rotary_dim: int, theta: float, device, scaling: RopeScaling | None = None):
    """float32 cos/sin ``[max_len, rotary_dim]`` built like ``model.py:66-92``
    (``inv_freq = theta^(-2i/rot)``, ``emb = cat(freqs, freqs)``); with
    ``scaling``, its frequencies, and angles in 64 bits (a float32 angle at
    position 2^20 is off by 2^-5)."""
    if scaling is not None:
        inv, mult = scaling.frequencies(rotary_dim, theta, device)
        a = torch.outer(torch.arange(max_len, device=device, dtype=torch.float64), inv)
        a = torch.cat((a, a), dim=-1)
        return (a.cos() * mult).float().contiguous(), (a.sin() * mult).float().contiguous()
    inv_freq = 1.0 / (theta ** (torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float32) / rotary_dim))
    t = torch.arange(max_len, device=device, dtype=torch.float32)
    freqs = torch.outer(t, inv_freq)
    emb = torch.cat((freqs, freqs), dim=-1)
    return emb.cos().contiguous(), emb.sin().contiguous()


def _bytes(t: torch.Tensor) -> torch.Tensor:
    """A float8 tensor as its bytes; any other as it is."""
    return t.view(torch.uint8) if t.element_size() == 1 else t


def _check_trees(cache) -> None:
    if getattr(cache, "k_scale", None) is not None or getattr(cache, "prefix", None) is not None:
        raise ValueError("drafted trees need a bf16 cache without shared prefixes.")


@dataclass
class SharedKV:
    """Prefixes that rows of a ``KVCache`` share (``KVCache.share``): per layer K/V ``[P,
    n_kv, longest, D]`` of the cache's kind, ``length [P]`` the prefixes' positions,
    ``of [slots]`` each slot's prefix (-1: none).  Indexed by slot like ``seqlen``."""

    k: list
    v: list
    length: torch.Tensor
    of: torch.Tensor
    k_scale: list | None = None
    v_scale: list | None = None

    @property
    def max_len(self) -> int:
        return int(self.k[0].shape[2])

    def layer(self, i: int, width: int) -> SharedPrefix:
        """Layer ``i``'s prefixes for a step over slots ``[0, width)``."""
        kv = KV(self.k[i], self.v[i]) if self.k_scale is None else QuantKV(self.k[i], self.v[i], self.k_scale[i],
                                                                           self.v_scale[i])
        return SharedPrefix(kv, self.length, self.of[:width])


@dataclass
class KVCache:
    """Preallocated bf16 K/V per layer ``[rows, n_kv, max_len, D]``, one write
    position per slot (``model.py:116-143``) and the attention workspace
    (zeroed once; the kernels leave its barrier counters zero).

    Slots and cache rows (``model.py:145-156, 196-214``): ``seqlen`` is
    indexed by slot, K/V by cache row, and ``row_map[slot]`` names the row.
    With ``remap`` off the map is the identity; a scheduler turns it on to
    keep live sequences in the low slots by swapping indices (never K/V), so
    a decode step can run at a narrow width.  A step of width ``w`` covers
    slots ``[0, w)``.

    With ``k_scale`` / ``v_scale`` the K/V are e4m3 codes with a power of two per
    position and head (``kernels.quant_cache``), half the bytes; with ``prefix``
    slots' sequences may begin with shared prefixes, ``seqlen`` then counting a
    slot's own positions.  Neither carries drafted trees.  ``attn_ws``: the
    workspace of a bf16 cache's steps (a quantised one's need none that is kept)."""

    k: list
    v: list
    seqlen: torch.Tensor
    max_len: int
    attn_ws: torch.Tensor = field(default=None)
    row_map: torch.Tensor = field(default=None)
    remap: bool = False
    k_scale: list | None = None
    v_scale: list | None = None
    prefix: SharedKV | None = None

    def __post_init__(self):
        if self.row_map is None:
            self.row_map = torch.arange(self.rows, device=self.seqlen.device, dtype=torch.int64)

    @property
    def rows(self) -> int:
        return int(self.k[0].shape[0])

    def slot_rows(self, width: int):
        """``(seqlen, row_map)`` views for a step over slots ``[0, width)``;
        ``row_map`` is None when the kernels may read row == slot."""
        if not 0 < width <= self.rows:
            raise ValueError(f"step width {width} outside the cache's {self.rows} slots.")
        rm = self.row_map[:width] if (self.remap or width != self.rows) else None
        return self.seqlen[:width], rm

    def swap_slots(self, i: int, j: int) -> None:
        """Exchange two slots: their row map entries and write positions."""
        if i == j:
            return
        if not self.remap:
            raise RuntimeError("swap_slots needs cache.remap: without the map the kernels read "
                               "cache row == slot, and a swap would read another sequence's K/V.")
        for t in (self.row_map, self.seqlen) + (() if self.prefix is None else (self.prefix.of,)):
            a = t[i].clone()
            t[i] = t[j]
            t[j] = a

    def reset_slot(self, slot: int) -> None:
        """Forget a slot's history so a new sequence can take it."""
        self.seqlen[slot] = 0
        if self.prefix is not None:
            self.prefix.of[slot] = -1

    @property
    def is_quantized(self) -> bool:
        return self.k_scale is not None

    def layer(self, i: int):
        """Layer ``i``'s ``KV`` or ``QuantKV``."""
        if self.k_scale is None:
            return KV(self.k[i], self.v[i])
        return QuantKV(self.k[i], self.v[i], self.k_scale[i], self.v_scale[i])

    def positions(self, width: int) -> torch.Tensor:
        """Where the next token of slots ``[0, width)`` stands in its sequence: behind
        its prefix and its own positions."""
        seqlen, p = self.seqlen[:width], self.prefix
        if p is None:
            return seqlen
        of = p.of[:width]
        n = p.length.shape[0]
        return seqlen + torch.where((of >= 0) & (of < n), p.length[of.clamp(0, n - 1)], 0)

    def quantized(self) -> "KVCache":
        """The same sequences in a quantised cache of their own (bf16 caches without
        prefixes)."""
        if self.is_quantized or self.prefix is not None:
            raise ValueError("quantized takes a bf16 cache without shared prefixes.")
        out = [quantize_kv(k, v, make_quant_kv(*k.shape, k.device)) for k, v in zip(self.k, self.v)]
        return KVCache([c.k for c in out], [c.v for c in out], self.seqlen.clone(), self.max_len, None,
                       self.row_map.clone(), self.remap, [c.k_scale for c in out], [c.v_scale for c in out])

    def dequantized(self) -> "KVCache":
        """The same sequences, as the codes stand for them, in a bf16 cache of their own."""
        if not self.is_quantized or self.prefix is not None:
            raise ValueError("dequantized takes a quantised cache without shared prefixes.")
        out = [dequantize_kv(self.layer(i)) for i in range(len(self.k))]
        rows, n_kv, max_len, d = self.k[0].shape
        return KVCache([c.k for c in out], [c.v for c in out], self.seqlen.clone(), self.max_len,
                       gqa_workspace(rows, n_kv, max_len, self.seqlen.device, d), self.row_map.clone(), self.remap)

    def share(self, rows, lengths) -> SharedKV:
        """Take the first ``lengths[p]`` positions of cache row ``rows[p]`` as prefix ``p``
        (copied: the rows are free again), held once for all slots that begin with it.
        Every slot begins with none; ``prefix.of[slot] = p`` with ``seqlen[slot]`` set to
        the slot's own positions (0 for a new sequence) puts one behind prefix ``p``.
        The model's rotary tables have to reach the longest prefix and a whole row
        (``max_len`` of both together): its steps refuse the cache else.
        Share before capturing a step: a graph captured earlier knows of no prefixes."""
        rows, lengths = [int(r) for r in rows], [int(n) for n in lengths]
        if self.prefix is not None:
            raise ValueError("the cache has shared prefixes already.")
        if len(rows) != len(lengths) or not rows:
            raise ValueError(f"share expects a length for each row, got {len(rows)} rows and {len(lengths)} lengths.")
        if any(not 0 <= r < self.rows for r in rows) or any(not 1 <= n <= self.max_len for n in lengths):
            raise ValueError(f"share: rows {rows} and lengths {lengths} for a cache of {self.rows} rows of {self.max_len}.")
        most = max(lengths)

        def take(layers):
            return None if layers is None else [t[rows, :, :most].contiguous() for t in layers]

        def codes(layers):  # (float8 tensors are indexed as the bytes they are)
            return None if layers is None else [t.view(torch.uint8)[rows, :, :most].contiguous().view(t.dtype)
                                                for t in layers]

        kv = codes if self.is_quantized else take
        dev = self.seqlen.device
        self.prefix = SharedKV(kv(self.k), kv(self.v), torch.tensor(lengths, device=dev, dtype=torch.int64),
                               torch.full((self.rows,), -1, device=dev, dtype=torch.int64), codes(self.k_scale),
                               codes(self.v_scale))
        return self.prefix

    def commit(self, path: torch.Tensor, accepted: torch.Tensor) -> None:
        """Keep an accepted branch of the nodes that ``forward_tree`` wrote behind
        slots ``[0, len(accepted))`` (``path`` / ``accepted`` as ``verify_tree``
        returns them for a tree that fits the cache, ``kernels.tree.fit_tree``):
        their K/V move together, in every layer, and the write positions advance
        past them.  Graph-safe; no host synchronisation."""
        _check_trees(self)
        seqlen, row_map = self.slot_rows(int(accepted.shape[0]))
        seqlen.copy_(commit_tree(self.k, self.v, seqlen, path, accepted, row_map=row_map))

    def snapshot(self, steps: int | None = None) -> dict:
        """Write positions, slot map and a copy of the K/V that the next
        ``steps`` decode steps can overwrite (all of it when ``steps`` is
        None); ``restore`` puts them back (``model.py:276-291``)."""
        lo, hi = 0, self.max_len
        if steps is not None:
            sl = self.seqlen.cpu()
            lo = int(sl.min()) if sl.numel() else 0
            hi = min(self.max_len, int(sl.max()) + int(steps) + 1) if sl.numel() else 0
        return {"seqlen": self.seqlen.clone(), "row_map": self.row_map.clone(), "remap": self.remap,
                "of": None if self.prefix is None else self.prefix.of.clone(), "span": (lo, hi),
                **{n: [_bytes(t)[:, :, lo:hi].clone() for t in ts] for n, ts in self._tensors().items()}}

    def _tensors(self) -> dict:
        names = ("k", "v", "k_scale", "v_scale") if self.is_quantized else ("k", "v")
        return {n: getattr(self, n) for n in names}

    def restore(self, snap: dict) -> None:
        self.seqlen.copy_(snap["seqlen"])
        self.row_map.copy_(snap["row_map"])
        self.remap = snap["remap"]
        if self.prefix is not None:
            self.prefix.of.fill_(-1) if snap["of"] is None else self.prefix.of.copy_(snap["of"])
        lo, hi = snap["span"]
        for n, ts in self._tensors().items():
            for dst, src in zip(ts, snap[n]):
                _bytes(dst)[:, :, lo:hi].copy_(src)


class SyntheticDecoder:
    def __init__(self, cfg: DecoderConfig, device, seed: int = 0, max_len: int = 4096 + 128,
                 fused_moe: bool = True, fused_o: bool = False, combine_next: bool = True,
                 o_in_moe: bool = False, prefetch_router: bool = True):
        self.cfg = cfg
        self.prefetch_router = prefetch_router
        self.fused_moe = fused_moe
        self.combine_next = combine_next
        self.fused_o = fused_o
        self.o_in_moe = o_in_moe
        self.device = torch.device(device)
        self.max_len = max_len
        c, dev, s = cfg, self.device, seed * 1000
        ones = lambda n: torch.ones(n, device=dev, dtype=torch.float32)
        self.layers = []
        for i in range(c.layers):
            qkv, qkv_a = synthetic.ternary_linear(c.qkv_rows, c.hidden, s + 10 * i + 1, dev)
            o, o_a = synthetic.ternary_linear(c.hidden, c.heads * c.head_dim, s + 10 * i + 2, dev)
            moe = synthetic.make_moe_layer(c.hidden, c.experts, c.inter, seed=s + 10 * i + 3, device=dev)
            self.layers.append(DecoderLayerWeights(qkv, qkv_a, o, o_a, ones(c.hidden), ones(c.hidden),
                                                   ones(c.head_dim), ones(c.head_dim), moe))
        lo, hi = c.lm_scale
        self.lm_head = synthetic.rtn4_table(c.vocab, c.hidden, c.rtn_group, s + 901, dev, lo, hi)
        self.embed = synthetic.rtn4_table(c.vocab, c.hidden, c.rtn_group, s + 902, dev, lo, hi)
        self.final_norm = ones(c.hidden)
        self.cos, self.sin = rope_tables(max_len, c.rotary_dim, c.rope_theta, dev, c.rope_scaling)
        self.flash_head = None
        self._pack_read_ahead()

    @classmethod
    def from_weights(cls, cfg: DecoderConfig, device, layers: list, embed: tuple, lm_head: tuple,
                     final_norm: torch.Tensor, max_len: int = 4096 + 128, fused_moe: bool = True,
                     fused_o: bool = False, combine_next: bool = True,
                     o_in_moe: bool = False, prefetch_router: bool = True) -> "SyntheticDecoder":
        """A decoder over given weights (``checkpoint.load_decoder``) instead of
        the seeded synthetic ones."""
        self = cls.__new__(cls)
        self.cfg = cfg
        self.fused_moe, self.fused_o, self.combine_next = fused_moe, fused_o, combine_next
        self.o_in_moe = o_in_moe
        self.prefetch_router = prefetch_router
        self.device = torch.device(device)
        self.max_len = max_len
        self.layers = list(layers)
        self.embed, self.lm_head, self.final_norm = embed, lm_head, final_norm
        self.cos, self.sin = rope_tables(max_len, cfg.rotary_dim, cfg.rope_theta, self.device, cfg.rope_scaling)
        self.flash_head = None
        self._pack_read_ahead()
        return self

    def _pack_read_ahead(self) -> None:
        """Lay out each layer's post-attention norm weights, QK-norm weights
        and router rows in one buffer (in that order, 256-byte aligned; the
        layer's tensors become views of it), which the previous layer's
        one-launch MoE kernel reads ahead into every XCD's L2 while it waits
        on its own hand-offs: bytes that are read at the start of the layer's
        launches and would otherwise come cold from HBM (the small ones first,
        so that a router larger than the read-ahead still leaves them in)."""
        self.read_ahead = []
        for i, L in enumerate(self.layers):
            parts = [L.post_ln, L.q_norm, L.k_norm, L.moe.gate_weight]
            offs, n = [], 0
            for t in parts:
                offs.append(n)
                n += -(-t.numel() * t.element_size() // 256) * 256
            buf = torch.empty(n, dtype=torch.uint8, device=L.post_ln.device)
            views = []
            for t, o in zip(parts, offs):
                v = buf[o:o + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
                v.copy_(t)
                views.append(v)
            moe = dataclasses.replace(L.moe, gate_weight=views[3])
            self.layers[i] = dataclasses.replace(L, post_ln=views[0], q_norm=views[1], k_norm=views[2], moe=moe)
            self.read_ahead.append(buf)

    def make_cache(self, batch: int, prefill_len: int, seed: int = 0, *, quantized: bool = False,
                   max_len: int | None = None) -> KVCache:
        """Cache rows filled with seeded N(0, 1) bf16 K/V for ``prefill_len``
        positions, of ``max_len`` (by default the model's); decoding then writes at
        ``prefill_len``.  ``quantized``: the same values in a quantised cache, never
        all of them in bf16."""
        c = self.cfg
        max_len = self.max_len if max_len is None else int(max_len)
        if not 1 <= max_len <= self.max_len:
            raise ValueError(f"make_cache: rows of {max_len} positions, the model has {self.max_len}.")
        shape = (batch, c.kv_heads, max_len, c.head_dim)

        def layer(i: int) -> KV:
            kv = KV(*(synthetic.randn_bf16(shape, 50_000 + j + seed * 97 + 2 * i, self.device) for j in range(2)))
            for t in kv:
                t[:, :, prefill_len:] = 0
            return kv

        if quantized:  # (one bf16 layer at a time beside the codes)
            layers = [quantize_kv(*layer(i), make_quant_kv(*shape, self.device)) for i in range(c.layers)]
        else:
            layers = [layer(i) for i in range(c.layers)]
        seqlen = torch.full((batch,), prefill_len, device=self.device, dtype=torch.int64)
        ws = None if quantized else gqa_workspace(batch, c.kv_heads, max_len, self.device, c.head_dim)
        names = ("k", "v", "k_scale", "v_scale") if quantized else ("k", "v")
        return KVCache(seqlen=seqlen, max_len=max_len, attn_ws=ws,
                       **{n: [kv[j] for kv in layers] for j, n in enumerate(names)})

    def _places(self, cache: KVCache, width: int):
        """What a step over slots ``[0, width)`` of a quantised cache, or of one with
        shared prefixes, needs in every layer: the new tokens' positions and, for a
        bf16 cache, the RoPE rows there.  None for any other cache."""
        if cache.prefix is None and not cache.is_quantized:
            return None
        if cache.prefix is not None and cache.prefix.max_len + cache.max_len > self.cos.shape[0]:
            raise ValueError(f"rotary tables of {self.cos.shape[0]} positions for prefixes of {cache.prefix.max_len} and "
                             f"rows of {cache.max_len}: give the model a larger max_len.")
        pos = cache.positions(width)
        if cache.is_quantized:
            return pos, None, None
        at = pos.clamp(0, self.cos.shape[0] - 1)
        return pos, self.cos[at], self.sin[at]

    def _cached_attention(self, i: int, qkv: torch.Tensor, cache: KVCache, seqlen: torch.Tensor, places, akw: dict):
        """Layer ``i``'s store and attention over a quantised cache or behind shared
        prefixes."""
        c, L = self.cfg, self.layers[i]
        pos, cos, sin = places
        kw = dict(num_heads=c.heads, num_kv_heads=c.kv_heads, head_dim=c.head_dim, rotary_dim=c.rotary_dim,
                  use_rope=akw["use_rope"], eps=c.eps, row_map=akw["row_map"])
        kv = cache.layer(i)
        if cache.prefix is None:
            return quant_attention(qkv, L.q_norm, L.k_norm, self.cos, self.sin, kv, seqlen, scale=akw["scale"],
                                   window=akw["window"], **kw)
        if cache.is_quantized:
            q = apply_qkv_quant(qkv, L.q_norm, L.k_norm, self.cos, self.sin, kv, seqlen, positions=pos, **kw)
        else:
            q = apply_qkv_decode(qkv, L.q_norm, L.k_norm, cos, sin, kv.k, kv.v, seqlen, use_qk_norm=True, **kw)
        kw = dict(row_map=akw["row_map"], scale=akw["scale"], window=akw["window"])
        return prefix_gqa_attn(q, kv, seqlen, cache.prefix.layer(i, qkv.shape[0]), **kw)

    def _layer(self, i: int, hidden: torch.Tensor, cache: KVCache, routing=None,
               qkv: torch.Tensor | None = None, fuse_next: bool = True, tree: torch.Tensor | None = None,
               places=None):
        """Layer ``i``; returns ``(y, next_qkv)``.  ``qkv``: this layer's input
        projection if an earlier launch already computed it.  ``next_qkv`` is
        layer ``i + 1``'s projection when the one-launch MoE kernel computed it
        from ``y`` (batch 1, ``fuse_next``), else None.  ``y`` is a
        ``PendingCombine`` where layer ``i + 1``'s QKV launch runs the MoE
        combine (``combine_next``, 17+ tokens); ``hidden`` may be one.
        ``tree [w, T]``: the parents of the ``w * T`` nodes that ``hidden``
        holds, instead of one token per slot.  ``places``: ``_places`` of the step."""
        c, L = self.cfg, self.layers[i]
        if isinstance(hidden, PendingCombine):  # the previous layer's MoE combine runs here
            hidden, qkv = ternary_gemv_combine(hidden, L.qkv, L.qkv_alpha, rms_weight=L.input_ln,
                                               rms_eps=c.eps)
        bsz = hidden.shape[0]
        if qkv is None:
            qkv = ternary_gemv(hidden, L.qkv, L.qkv_alpha, rms_weight=L.input_ln, rms_eps=c.eps)
        window, use_rope = c.layer_attention(i)
        akw = dict(num_heads=c.heads, num_kv_heads=c.kv_heads, head_dim=c.head_dim,
                   rotary_dim=c.rotary_dim, eps=c.eps, scale=c.head_dim ** -0.5, window=window,
                   use_rope=use_rope)
        seqlen, row_map = cache.slot_rows(bsz if tree is None else tree.shape[0])
        akw["row_map"] = row_map
        if (bsz == 1 and tree is None and places is None and self.fused_o
                and o_projection_supported(1, c.heads, c.kv_heads, c.head_dim, cache.max_len, window, c.hidden)):
            # attention and its output projection in one launch (measured: no
            # faster than two launches at 4096 positions -- the grid barrier
            # and the tail cost what the second launch does -- so off by default)
            _, o = decode_attention(qkv, L.q_norm, L.k_norm, self.cos, self.sin, cache.k[i], cache.v[i],
                                    seqlen, cache.attn_ws, o_linear=(L.o, L.o_alpha), **akw)
        else:
            if places is not None:
                attn = self._cached_attention(i, qkv, cache, seqlen, places, akw)
            elif tree is None:
                attn = decode_attention(qkv, L.q_norm, L.k_norm, self.cos, self.sin, cache.k[i], cache.v[i],
                                        seqlen, cache.attn_ws, **akw)
            else:
                scale, window = akw.pop("scale"), akw.pop("window")
                q = apply_qkv_tree(qkv.view(*tree.shape, -1), L.q_norm, L.k_norm, self.cos, self.sin, cache.k[i],
                                   cache.v[i], seqlen, tree, **akw)
                attn = tree_attention(q, cache.k[i], cache.v[i], seqlen, tree, row_map=row_map, scale=scale,
                                      window=window)
            # o_in_moe: at batch 1 the XCD-split MoE launch computes the output
            # projection itself (same bits; measured 1,294 against 1,306 tok/s
            # with the separate launch, so off by default)
            o_moe = (bsz == 1 and self.o_in_moe and self.fused_moe and fused_supported(L.moe, c.top_k, hidden)
                     and fused_form(L.moe, c.top_k) == 1 and c.heads * c.head_dim == c.hidden
                     and L.o_alpha.dtype == L.moe.up_gate_alpha.dtype)
            o = None if o_moe else ternary_gemv(attn.reshape(bsz, -1), L.o, L.o_alpha)
        next_qkv = None
        if bsz == 1 and self.fused_moe and fused_supported(L.moe, c.top_k, hidden):
            # add + RMSNorm + router + experts + combine (+ the next layer's
            # RMS-folded QKV projection) in one launch
            nl = None
            if fuse_next and i + 1 < c.layers and self.layers[i + 1].qkv_alpha.dtype == L.moe.up_gate_alpha.dtype:
                n = self.layers[i + 1]
                nl = (n.qkv, n.qkv_alpha, n.input_ln, c.eps)
            # the next layer's norm weights and router rows are read ahead
            # into the caches while this launch waits for h
            pf = self.read_ahead[i + 1] if self.prefetch_router and i + 1 < c.layers else None
            out = moe_fused(hidden, L.moe, c.top_k, add=o, norm_weight=L.post_ln, eps=c.eps,
                            next_linear=nl,
                            o_linear=None if o is not None else (attn.reshape(1, -1), L.o, L.o_alpha),
                            prefetch=pf)
            y, ids = out[0], out[1]
            if nl is not None:
                next_qkv = out[3]
        else:
            # add + RMSNorm + router + dispatch in one launch from 4 tokens,
            # then the grouped experts
            defer = (self.combine_next and fuse_next and i + 1 < c.layers
                     and combine_gemv_supported(bsz, c.top_k, self.layers[i + 1].qkv))
            y, ids = moe_layer(hidden, L.moe, c.top_k, L.post_ln, c.eps, add=o.reshape(hidden.shape),
                               defer_combine=defer)
        if routing is not None:
            routing.append(ids)
        return y, next_qkv

    def layer_step(self, i: int, hidden: torch.Tensor, cache: KVCache, routing=None) -> torch.Tensor:
        """Layer ``i`` on its own (its QKV projection computed here)."""
        return self._layer(i, hidden, cache, routing, fuse_next=False, places=self._places(cache, hidden.shape[0]))[0]

    def forward(self, input_ids: torch.Tensor, cache: KVCache, routing: list | None = None) -> torch.Tensor:
        """One decode step for ``input_ids [w]`` over cache slots ``[0, w)``;
        returns bf16 logits ``[w, vocab]``.  ``routing``, if a list, receives
        each layer's expert ids."""
        width = int(input_ids.numel())
        cache.slot_rows(width)
        hidden = self.embed_tokens(input_ids.reshape(-1))
        qkv = None
        places = self._places(cache, width)
        for i in range(self.cfg.layers):
            hidden, qkv = self._layer(i, hidden, cache, routing, qkv, places=places)
        cache.seqlen[:width].add_(1)
        return self.head(hidden)

    def forward_tree(self, tokens: torch.Tensor, parents: torch.Tensor, cache: KVCache,
                     routing: list | None = None) -> torch.Tensor:
        """The model over a tree of drafted tokens per row: ``tokens [w, T]``, node
        0 each row's last token, ``parents [w, T]`` (``kernels.tree``) over cache
        slots ``[0, w)``.  Writes the nodes' K/V at ``seqlen .. seqlen + T - 1``
        without advancing ``seqlen`` (``KVCache.commit`` does) and returns bf16
        logits ``[w, T, vocab]``; a chain's are those of as many decode steps up to
        rounding, from the head that such steps use: at one row the FlashHead, if
        one is attached, node by node.  Padding's logits say nothing."""
        w, t = tokens.shape
        _check_trees(cache)
        cache.slot_rows(w)
        parents = check_tree("forward_tree", parents, w, t)  # (once, not in each layer)
        hidden = self.embed_tokens(tokens.reshape(-1))  # (padding's ids are clamped to the table)
        qkv = None
        for i in range(self.cfg.layers):
            hidden, qkv = self._layer(i, hidden, cache, routing, qkv, tree=parents)
        if self.flash_head is None or w > 1:
            return self.head(hidden).view(w, t, -1)
        # (rows of their own, 16-byte aligned, which the next call leaves alone)
        v = self.cfg.vocab
        logits = torch.empty(t, -(-v // 8) * 8, device=hidden.device, dtype=torch.bfloat16)[:, :v]
        hidden = rms_norm(hidden, self.final_norm, self.cfg.eps)
        for i in range(t):
            self.flash_head(hidden[i:i + 1], out=logits[i])
        return logits.unsqueeze(0)

    def embed_tokens(self, input_ids: torch.Tensor) -> torch.Tensor:
        w, sc, bs = self.embed
        return rtn4_embedding(input_ids, w, sc, bs, group_size=self.cfg.rtn_group).to(torch.bfloat16)

    def head(self, hidden: torch.Tensor) -> torch.Tensor:
        """Final RMSNorm and the RTN4 lm_head: bf16 logits ``[B, vocab]``
        (at batch 1 through the FlashHead when one is attached: -inf outside
        the probed clusters and forced tokens, model.py:874-886)."""
        hidden = rms_norm(hidden, self.final_norm, self.cfg.eps)
        if self.flash_head is not None and hidden.shape[0] == 1:
            return self.flash_head(hidden).reshape(1, -1)
        w, sc, bs = self.lm_head
        return rtn4_gemv(hidden, w, sc, bs, group_size=self.cfg.rtn_group)

    def greedy_step(self, ids: torch.Tensor, cache: KVCache) -> torch.Tensor:
        """forward + argmax, writing the next ids back into ``ids`` (graph-safe)."""
        logits = self.forward(ids, cache)
        greedy_argmax(logits, out=ids)
        return logits

    def decode_bytes(self, batch: int, kv_len: int) -> int:
        """Algorithmic HBM bytes of one decode step: weights touched once; the
        experts a step touches counted as the expected number of distinct
        experts among ``batch`` rows of top-k picks under uniform routing,
        E (1 - (1 - k/E)^batch) (k at batch 1, all E at large batches); the
        KV read for every row over the positions each layer attends (the last
        ``sliding_window`` on sliding layers)."""
        c = self.cfg
        lay = (c.qkv_rows + c.hidden) * c.hidden // 4 + (c.qkv_rows + c.hidden) * 2
        router = c.experts * c.hidden * 2
        expert = (3 * c.inter * c.hidden) // 4 + (2 * c.inter + c.hidden) * 2
        hit = c.experts * (1.0 - (1.0 - c.top_k / c.experts) ** batch)
        experts = int(round(hit * expert))
        kv = 0
        for i in range(c.layers):
            window, _ = c.layer_attention(i)
            span = min(kv_len, window) if window else kv_len
            kv += batch * 2 * c.kv_heads * span * c.head_dim * 2
        head = c.vocab * c.hidden // 2 + 2 * c.vocab * (c.hidden // c.rtn_group) * 2
        return c.layers * (lay + router + experts) + kv + head
