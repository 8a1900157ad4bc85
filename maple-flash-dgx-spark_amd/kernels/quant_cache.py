"""A quantised KV cache, and attention over it and over shared prefixes.

A ``QuantKV`` holds, per (row, KV head, position) and for K and V each,
``head_dim`` e4m3 codes and one power of two (e8m0): the least ``2^e`` with which
the largest finite value is at most ``448 * 2^e`` (``e`` in -126 .. 119), so
``head_dim + 1`` bytes where a bf16 cache holds ``2 * head_dim``.  A code is off by
at most 2^-4 of its value (2^-10 of the scale for small ones); values that are not
finite become NaN.  ``apply_qkv_quant`` writes a step's tokens, ``quantize_kv`` whole
prompts, ``dequantize_kv`` reads positions back, ``quant_gqa_attn`` attends;
``quant_attention`` is a step's ``apply_qkv_quant`` and ``quant_gqa_attn`` together.

A ``SharedPrefix`` holds the K/V with which several rows' sequences begin: row
``b``'s is the first ``length[of[b]]`` positions of prefix ``of[b]`` (any value that
is no prefix's index: none), then the row's own cached positions 0 .. ``seqlen[b]``.
``prefix_gqa_attn`` reads a long prefix once for all of its rows, in a bf16 (``KV``) or a
quantised cache.

No reference counterpart: its cache is bf16 with a row to a sequence
(``src/maple_run/model.py:116-291``), and its QK-norm, RoPE, K/V store and GQA
(``src/maple_run/kernels/decode_attn.py:362-592``) are these for such a cache.
``seqlen[b]`` is the index of the row's last own token, as there; here a negative
one marks a row without any (nothing is stored, Q is 0), and a token past the
cache's end is not stored.  ``row_map`` (slot -> cache row) names each cache row that
is written once.  All of these can be captured into a graph.
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from .. import _lib
from .tree import _FAR, _call, _device, _positions

CODE = torch.float8_e4m3fn
SCALE = torch.float8_e8m0fnu

_contiguous, _ptr = torch.Tensor.is_contiguous, torch.Tensor.data_ptr


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*sizes: int) -> int:
    return int(_lib.load().ma_cache_attn_workspace_bytes(*sizes))


class KV(NamedTuple):
    """A bf16 cache: ``k`` / ``v [rows, n_kv, max_len, head_dim]``."""

    k: torch.Tensor
    v: torch.Tensor


class QuantKV(NamedTuple):
    """A quantised cache: e4m3 ``k`` / ``v [rows, n_kv, max_len, head_dim]`` and e8m0
    ``k_scale`` / ``v_scale [rows, n_kv, max_len]``."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


class SharedPrefix(NamedTuple):
    """``cache``: a ``KV`` or ``QuantKV`` of P rows, a prefix each; ``length [P]``: their
    positions; ``of [B]``: each batch row's prefix (-1: none)."""

    cache: KV | QuantKV
    length: torch.Tensor
    of: torch.Tensor


def make_quant_kv(rows: int, num_kv_heads: int, max_len: int, head_dim: int, device) -> QuantKV:
    """An empty quantised cache (all values 0)."""
    shape = (rows, num_kv_heads, max_len)
    return QuantKV(*(torch.zeros(*shape, head_dim, device=device, dtype=CODE) for _ in range(2)),
                   *(torch.full(shape, 1, device=device, dtype=torch.uint8).view(SCALE) for _ in range(2)))


def _check_cache(what: str, cache, bsz: int | None, row_map):
    """The caches' shape ``[rows, n_kv, max_len, head_dim]``."""
    k, v = cache[0], cache[1]
    shape = k.shape
    if len(shape) != 4 or v.shape != shape:
        raise ValueError(f"{what}: K {tuple(shape)} and V {tuple(v.shape)} caches, "
                         "expected [rows, n_kv, max_len, head_dim] twice.")
    want = torch.bfloat16
    if len(cache) == 4:
        want, k_scale, v_scale = CODE, cache[2], cache[3]
        if k_scale.dtype != SCALE or v_scale.dtype != SCALE:
            raise TypeError(f"{what}: scales must be {SCALE}; got {k_scale.dtype} and {v_scale.dtype}.")
        if k_scale.shape != v_scale.shape or k_scale.shape != shape[:3]:
            raise ValueError(f"{what}: scales {tuple(k_scale.shape)} and {tuple(v_scale.shape)} for a cache {tuple(shape)}.")
    if k.dtype != want or v.dtype != want:
        raise TypeError(f"{what}: K and V caches of {k.dtype} and {v.dtype}, expected {want}.")
    if not all(map(_contiguous, cache)):
        raise ValueError(f"{what}: the cache must be contiguous.")
    if row_map is None and bsz is not None and shape[0] != bsz:
        raise ValueError(f"KV cache batch {shape[0]} != {what} batch {bsz}.")
    return shape


def _quant(what: str, cache) -> None:
    if not isinstance(cache, QuantKV):
        raise TypeError(f"{what} takes a QuantKV, got {type(cache).__name__}.")


def _window(window: int | None) -> int:
    if window is None:
        return 0
    if window < 1:
        raise ValueError(f"window must be positive, got {window}.")
    return min(window, _FAR)  # (past every position; more would wrap in 64 bits)


def _projection(what: str, qkv, q_weight, k_weight, cos_table, sin_table, cache, seqlen, positions, row_map, num_heads,
                num_kv_heads, head_dim, rotary_dim, use_rope, eps):
    """The checks of a token's projection and cache, the device, and the arguments from qkv to
    the cache's sizes (the last item: the tensors that they point to)."""
    _quant(what, cache)
    if qkv.ndim != 2 or qkv.dtype != torch.bfloat16:
        raise ValueError(f"{what} expects bf16 qkv [B, qkv], got {qkv.dtype} {tuple(qkv.shape)}.")
    bsz, width = qkv.shape
    if width != (num_heads + 2 * num_kv_heads) * head_dim:
        raise ValueError(f"qkv rows of {width}, expected {(num_heads + 2 * num_kv_heads) * head_dim}.")
    ldb, one = qkv.stride()
    if one != 1:
        raise ValueError(f"{what} needs a row-contiguous qkv.")
    rows, n_kv, max_len, d = _check_cache(what, cache, bsz, row_map)
    if n_kv != num_kv_heads or d != head_dim:
        raise ValueError(f"{what}: cache {tuple(cache.k.shape)} for {num_kv_heads} KV heads of {head_dim}.")
    more, qw, kw, c, s = [], None, None, None, None
    w_dt = dt = ld = n_pos = 0
    if q_weight is not None or k_weight is not None:
        if q_weight is None or k_weight is None:
            raise ValueError("q_weight and k_weight go together.")
        if q_weight.dtype != k_weight.dtype:
            raise TypeError("q_norm and k_norm weights must share a dtype.")
        if q_weight.numel() != head_dim or k_weight.numel() != head_dim:
            raise ValueError(f"norm weights need {head_dim} entries.")
        w_dt = _lib.dtype_code(q_weight, "q_weight")
        more = [q_weight.contiguous(), k_weight.contiguous()]
        qw, kw = more[0].data_ptr(), more[1].data_ptr()
    rot = rotary_dim if use_rope else 0
    if rot != 0:
        shape, strides = cos_table.shape, cos_table.stride()
        if (len(shape) != 2 or sin_table.shape != shape or sin_table.stride() != strides or strides[1] != 1
                or sin_table.dtype != cos_table.dtype):
            raise ValueError("cos and sin tables must share dtype and layout, rows contiguous.")
        n_pos, ld = shape[0], strides[0]
        if n_pos < 1 or shape[1] < rot:
            raise ValueError(f"tables {tuple(shape)} for a rotary_dim of {rot}.")
        dt = _lib.dtype_code(cos_table, "cos_table")
        more += [cos_table, sin_table]
        c, s = cos_table.data_ptr(), sin_table.data_ptr()
    sl = _positions("seqlen", seqlen, bsz)
    at = rm = None
    if positions is not None:
        more.append(_positions("positions", positions, bsz))
        at = more[-1].data_ptr()
    if row_map is not None:
        more.append(_positions("row_map", row_map, bsz))
        rm = more[-1].data_ptr()
    idx = _device(what, qkv, *cache, sl, *more)
    more.append(sl)
    return idx, (qkv.data_ptr(), ldb if bsz > 1 else width, bsz, num_heads, num_kv_heads, head_dim, qw, kw, w_dt, c, s, dt, ld,
                 n_pos, rot, eps, sl.data_ptr(), at, rm, *map(_ptr, cache), rows, max_len), more


def apply_qkv_quant(
    qkv: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    cos_table: torch.Tensor,
    sin_table: torch.Tensor,
    cache: QuantKV,
    seqlen: torch.Tensor,
    *,
    positions: torch.Tensor | None = None,
    row_map: torch.Tensor | None = None,
    num_heads: int,
    num_kv_heads: int,
    head_dim: int,
    rotary_dim: int,
    use_rope: bool = True,
    eps: float = 1e-6,
) -> torch.Tensor:
    """QK RMSNorm + RoPE + quantising store of K/V at ``seqlen``; returns Q ``[B, H,
    1, D]`` bf16.

    ``qkv [B, (H + 2 Hkv) D]`` bf16; ``q_weight`` / ``k_weight`` both None: no norm.
    The tables ``[n_pos, >= rotary_dim]`` are read at ``positions [B]``, by default
    ``seqlen`` (behind a shared prefix a token's position is further on).  K is
    rounded to bf16, as ``apply_qkv_decode`` stores it, and then quantised."""
    idx, args, _keep = _projection("apply_qkv_quant", qkv, q_weight, k_weight, cos_table, sin_table, cache, seqlen, positions,
                                   row_map, num_heads, num_kv_heads, head_dim, rotary_dim, use_rope, eps)
    out = qkv.new_empty(qkv.shape[0], num_heads, 1, head_dim)
    _call(idx, "ma_quant_qkv", *args, out.data_ptr())
    return out


def quantize_kv(
    k: torch.Tensor,
    v: torch.Tensor,
    cache: QuantKV,
    *,
    start: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    row_map: torch.Tensor | None = None,
) -> QuantKV:
    """Quantise ``k`` / ``v [B, n_kv, T, D]`` (bf16, the last dim contiguous) into the
    cache's positions ``start[b] ..`` (0 by default), of row ``b`` the first
    ``lengths[b]`` (all by default); everything else is left as it was.  Returns the
    cache."""
    _quant("quantize_kv", cache)
    if k.ndim != 4 or v.shape != k.shape:
        raise ValueError(f"quantize_kv expects k and v [B, n_kv, T, D], got {tuple(k.shape)} and {tuple(v.shape)}.")
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise TypeError(f"quantize_kv takes bf16 k and v; got {k.dtype} and {v.dtype}.")
    bsz, n_kv, t, d = k.shape
    rows, c_kv, max_len, c_d = _check_cache("quantize_kv", cache, bsz, row_map)
    if (c_kv, c_d) != (n_kv, d):
        raise ValueError(f"quantize_kv: cache {tuple(cache.k.shape)} for {n_kv} KV heads of {d}.")
    k_s, v_s = k.stride(), v.stride()
    if k_s[3] != 1 or v_s[3] != 1:
        raise ValueError("quantize_kv needs contiguous rows of k and v.")
    more, at = [], []
    for name, x in (("start", start), ("lengths", lengths), ("row_map", row_map)):
        if x is not None:
            more.append(_positions(name, x, bsz))
        at.append(None if x is None else more[-1].data_ptr())
    idx = _device("quantize_kv", k, v, *cache, *more)
    _call(
        idx, "ma_quant_kv",
        k.data_ptr(), *k_s[:3], v.data_ptr(), *v_s[:3], bsz, t, n_kv, d, *at,
        *map(_ptr, cache), rows, max_len,
    )
    return cache


def dequantize_kv(cache: QuantKV, length: int | None = None, *, row_map: torch.Tensor | None = None) -> KV:
    """The first ``length`` positions (all by default) of the cache's rows, or of the
    rows that ``row_map`` names, as bf16 ``[B, n_kv, length, D]``."""
    _quant("dequantize_kv", cache)
    rows, n_kv, max_len, d = _check_cache("dequantize_kv", cache, None, None)
    length = max_len if length is None else int(length)
    if not 0 <= length <= max_len:
        raise ValueError(f"dequantize_kv: {length} positions of a cache of {max_len}.")
    rm = None if row_map is None else _positions("row_map", row_map, row_map.numel())
    idx = _device("dequantize_kv", *cache, *(() if rm is None else (rm,)))
    shape = (rows if rm is None else rm.numel(), n_kv, length, d)
    k = cache.k.new_empty(*shape, dtype=torch.bfloat16)
    out = KV(k, torch.empty_like(k))
    _call(
        idx, "ma_dequant_kv",
        *map(_ptr, cache), rows, max_len, shape[0], length, n_kv, d, _lib.ptr(rm), out.k.data_ptr(),
        out.v.data_ptr(),
    )
    return out


_NO_PREFIX = (None,) * 4


def _attend(what: str, q: torch.Tensor, cache, seqlen: torch.Tensor, prefix: SharedPrefix | None, row_map, scale: float,
            window: int | None, once: bool | None = None) -> torch.Tensor:
    if q.ndim != 4 or q.shape[2] != 1 or q.dtype != torch.bfloat16:
        raise ValueError(f"{what} expects bf16 q [B, H, 1, D], got {q.dtype} {tuple(q.shape)}.")
    bsz, n_q, _, head_dim = q.shape
    rows, n_kv, max_len, d = _check_cache(what, cache, bsz, row_map)
    if d != head_dim:
        raise ValueError(f"{what}: cache {tuple(cache.k.shape)} for heads of {head_dim}.")
    if n_kv < 1 or n_q % n_kv != 0:
        raise ValueError(f"n_q={n_q} not divisible by n_kv={n_kv}.")
    window = _window(window)
    sl = _positions("seqlen", seqlen, bsz)
    more = []
    rm = None
    if row_map is not None:
        more.append(_positions("row_map", row_map, bsz))
        rm = more[-1].data_ptr()
    quant = len(cache) == 4
    shared, n_pre, pre_max, p_len, p_of = _NO_PREFIX, 0, 0, None, None
    if prefix is not None:
        if type(prefix.cache) is not type(cache):
            raise TypeError(f"{what}: a {type(cache).__name__} cache behind a {type(prefix.cache).__name__} prefix.")
        n_pre, p_kv, pre_max, p_d = _check_cache(what, prefix.cache, None, None)
        if (p_kv, p_d) != (n_kv, d):
            raise ValueError(f"{what}: prefixes {tuple(prefix.cache.k.shape)} for {n_kv} KV heads of {d}.")
        length, of = _positions("length", prefix.length, n_pre), _positions("of", prefix.of, bsz)
        more += [*prefix.cache, length, of]
        shared = (*map(_ptr, prefix.cache), *(() if quant else (None, None)))
        p_len, p_of = length.data_ptr(), of.data_ptr()
        if pre_max == 0:
            n_pre = 0
    idx = _device(what, q, *cache, sl, *more)
    if not q.is_contiguous():
        q = q.contiguous()
    out = torch.empty_like(q)
    form = -1 if once is None else int(once)
    nbytes = _workspace_bytes(bsz, n_q, n_kv, head_dim, max_len, n_pre, pre_max, window, quant, form)
    # scratch of this call alone: the allocator keeps it to this stream, a
    # captured graph to its own pool
    ws = q.new_empty(nbytes // 2) if nbytes else None
    _call(
        idx, "ma_cache_attn",
        q.data_ptr(), bsz, n_q, n_kv, head_dim, *map(_ptr, cache), *(() if quant else (None, None)), rows, max_len,
        sl.data_ptr(), rm, *shared, n_pre, pre_max, p_len, p_of, form, window, scale, out.data_ptr(), _lib.ptr(ws), nbytes,
    )
    return out


def quant_gqa_attn(
    q: torch.Tensor,
    cache: QuantKV,
    seqlen: torch.Tensor,
    *,
    row_map: torch.Tensor | None = None,
    scale: float,
    window: int | None = None,
) -> torch.Tensor:
    """GQA attention for ``q_len=1`` over a quantised cache: ``q [B, H, 1, D]`` bf16
    over positions 0 .. ``seqlen[b]`` (the last ``window`` of them), as
    ``decode_gqa_attn`` over the values that the codes stand for; a row without a
    token (``seqlen[b] < 0``) gives 0.  ``head_dim`` 64 or 128, at most 16 query
    heads to a KV head."""
    _quant("quant_gqa_attn", cache)
    return _attend("quant_gqa_attn", q, cache, seqlen, None, row_map, scale, window)


def quant_attention(
    qkv: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    cos_table: torch.Tensor,
    sin_table: torch.Tensor,
    cache: QuantKV,
    seqlen: torch.Tensor,
    *,
    positions: torch.Tensor | None = None,
    row_map: torch.Tensor | None = None,
    num_heads: int,
    num_kv_heads: int,
    head_dim: int,
    rotary_dim: int,
    use_rope: bool = True,
    eps: float = 1e-6,
    scale: float,
    window: int | None = None,
) -> torch.Tensor:
    """``apply_qkv_quant`` and then ``quant_gqa_attn`` with one launch less, as
    ``decode_attention`` is for a bf16 cache: the same codes stored, the attention output
    ``[B, H, 1, D]`` (its sums in another order)."""
    window = _window(window)
    idx, args, _keep = _projection("quant_attention", qkv, q_weight, k_weight, cos_table, sin_table, cache, seqlen, positions,
                                   row_map, num_heads, num_kv_heads, head_dim, rotary_dim, use_rope, eps)
    out = qkv.new_empty(qkv.shape[0], num_heads, 1, head_dim)
    nbytes = _workspace_bytes(qkv.shape[0], num_heads, num_kv_heads, head_dim, args[-1], 0, 0, window, True, -1)
    ws = qkv.new_empty(nbytes // 2) if nbytes else None  # (as in _attend)
    _call(idx, "ma_quant_attn", *args, window, scale, out.data_ptr(), _lib.ptr(ws), nbytes)
    return out


def prefix_gqa_attn(
    q: torch.Tensor,
    cache: KV | QuantKV,
    seqlen: torch.Tensor,
    prefix: SharedPrefix,
    *,
    row_map: torch.Tensor | None = None,
    scale: float,
    window: int | None = None,
    once: bool | None = None,
) -> torch.Tensor:
    """GQA attention for ``q_len=1`` over rows whose sequences begin with shared
    prefixes: ``q [B, H, 1, D]`` bf16 over prefix ``of[b]`` and then the row's own
    positions 0 .. ``seqlen[b]`` (none where that is negative), the last ``window`` of
    both together.  The prefix is of the cache's kind.

    ``once``: each prefix is read once for all of its rows (True; not under a window, nor
    for more than 64 prefixes), or by each row with its own positions (False).  By
    default as is faster for the caches' sizes, which the host knows: a caller whose
    prefixes are much shorter than their cache, or on whose longest one most rows
    stand, may know better."""
    if not isinstance(cache, (KV, QuantKV)):
        raise TypeError(f"prefix_gqa_attn takes a KV or a QuantKV, got {type(cache).__name__}.")
    return _attend("prefix_gqa_attn", q, cache, seqlen, prefix, row_map, scale, window, once)
