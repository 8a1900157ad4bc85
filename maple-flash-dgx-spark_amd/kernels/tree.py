"""Decoding with a tree of drafted tokens per row.

A draft proposes, behind a row's last token, a tree of tokens; one pass of the
model scores them all and the branch that the target's law accepts is kept.  Per
layer ``apply_qkv_tree`` then ``tree_attention``, on the logits ``verify_tree``,
and ``commit_tree`` on the cache (``model.SyntheticDecoder.tree_step`` runs
them).  No reference counterpart: its decode step takes one token per row
(``src/maple_run/kernels/decode_attn.py:362-592``, whose QK-norm, RoPE, K/V
store and GQA these are for several, and ``src/maple_run/kernels/sampler.py``,
whose law the verification keeps).

The tree is ``parents [B, T]``, ``T <= 64``, on the device: node 0 is the row's
last token (its K/V not yet cached) with parent -1, any other node's parent comes
before it (``0 <= parents[b, i] < i``).  A node with any other parent, and all
below it, is padding; a row whose entry 0 is not -1 has no sequence.  Node ``i``
is cached at ``seqlen[b] + i`` and stands at position ``seqlen[b] + depth``.  Row
``b`` needs ``seqlen[b] + T <= max_len``; nodes past the cache's end are neither
stored nor attended.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from .. import _lib
from .decode_attn import _check_rows, _i64
from .sampler import _check

MAX_NODES = 64


def _check_tree(parents: torch.Tensor, bsz: int, nodes: int, device: torch.device, what: str) -> torch.Tensor:
    if not 1 <= nodes <= MAX_NODES:
        raise ValueError(f"{what}: a tree has 1 to {MAX_NODES} nodes, got {nodes}.")
    if parents.shape != (bsz, nodes):
        raise ValueError(f"{what}: parents is {tuple(parents.shape)}, expected {(bsz, nodes)}.")
    if parents.dtype != torch.int32:
        if parents.dtype != torch.int64:
            raise TypeError(f"{what}: parents must be int32 or int64; got {parents.dtype}.")
        parents = parents.to(torch.int32)
    _same_device(what, device, parents)
    return parents.contiguous()


def _same_device(what: str, device: torch.device, *tensors) -> None:
    if device.type != "cuda":
        raise RuntimeError(f"{what} requires CUDA tensors.")
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: tensors on {t.device} and {device}.")


def _check_cache(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor, n_kv: int, head_dim: int) -> None:
    if k_cache.ndim != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"{what}: K {tuple(k_cache.shape)} and V {tuple(v_cache.shape)} caches, "
                         "expected [rows, n_kv, max_len, head_dim] twice.")
    if k_cache.shape[1] != n_kv or k_cache.shape[3] != head_dim:
        raise ValueError(f"{what}: cache {tuple(k_cache.shape)} for {n_kv} KV heads of {head_dim}.")


def apply_qkv_tree(
    qkv: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    cos_table: torch.Tensor,
    sin_table: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    seqlen: torch.Tensor,
    parents: torch.Tensor,
    *,
    row_map: torch.Tensor | None = None,
    num_heads: int,
    num_kv_heads: int,
    head_dim: int,
    rotary_dim: int,
    use_rope: bool = True,
    interleaved: bool = False,
    eps: float = 1e-6,
) -> torch.Tensor:
    """QK RMSNorm + rotary positions + K/V store of a tree's nodes; returns Q
    ``[B, T, H, D]`` (0 for padding).

    ``qkv [B, T, (H + 2 Hkv) D]`` bf16.  ``q_weight`` / ``k_weight`` both None:
    no norm.  The tables ``[n_pos, >= rotary_dim]`` (``model.rope_tables``, in any
    scaling) are read at each node's position; ``interleaved`` turns dims
    ``2i, 2i + 1`` together instead of ``i, i + rotary_dim / 2``."""
    if qkv.ndim != 3 or qkv.dtype != torch.bfloat16:
        raise ValueError(f"apply_qkv_tree expects bf16 qkv [B, T, qkv], got {qkv.dtype} {tuple(qkv.shape)}.")
    bsz, nodes, width = qkv.shape
    if width != (num_heads + 2 * num_kv_heads) * head_dim:
        raise ValueError(f"qkv rows of {width}, expected {(num_heads + 2 * num_kv_heads) * head_dim}.")
    if width > 1 and qkv.stride(2) != 1:
        raise ValueError("apply_qkv_tree needs a row-contiguous qkv.")
    _check_rows("qkv", bsz, k_cache, v_cache, seqlen, row_map)
    _check_cache("apply_qkv_tree", k_cache, v_cache, num_kv_heads, head_dim)
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight go together.")
    if q_weight is not None:
        if q_weight.dtype != k_weight.dtype:
            raise TypeError("q_norm and k_norm weights must share a dtype.")
        if q_weight.numel() != head_dim or k_weight.numel() != head_dim:
            raise ValueError(f"norm weights need {head_dim} entries.")
        q_weight, k_weight = q_weight.reshape(-1).contiguous(), k_weight.reshape(-1).contiguous()
    c = s = None
    dt = ld = n_pos = 0
    if use_rope and rotary_dim > 0:
        c, s = cos_table, sin_table
        if c.ndim != 2 or s.shape != c.shape or s.dtype != c.dtype or s.stride() != c.stride() or c.stride(1) != 1:
            raise ValueError("cos and sin tables must share dtype and layout, rows contiguous.")
        if c.shape[0] < 1 or c.shape[1] < rotary_dim:
            raise ValueError(f"tables {tuple(c.shape)} for a rotary_dim of {rotary_dim}.")
        dt, ld, n_pos = _lib.dtype_code(c, "cos_table"), c.stride(0), int(c.shape[0])
    dev = qkv.device
    parents = _check_tree(parents, bsz, nodes, dev, "apply_qkv_tree")
    sl, rm = _i64(seqlen), _i64(row_map)
    _same_device("apply_qkv_tree", dev, k_cache, v_cache, sl, rm, q_weight, k_weight, c, s)
    out = torch.empty(bsz, nodes, num_heads, head_dim, device=dev, dtype=torch.bfloat16)
    with torch.cuda.device(dev):
        _lib.call(
            "ma_tree_qkv",
            _lib.ptr(qkv), qkv.stride(0), qkv.stride(1), bsz, nodes, num_heads, num_kv_heads, head_dim,
            _lib.ptr(q_weight), _lib.ptr(k_weight), 0 if q_weight is None else _lib.dtype_code(q_weight, "q_weight"),
            _lib.ptr(c), _lib.ptr(s), dt, ld, n_pos, int(rotary_dim) if c is not None else 0,
            0 if c is None else (2 if interleaved else 1), float(eps), _lib.ptr(sl), _lib.ptr(parents), _lib.ptr(rm),
            _lib.ptr(k_cache), _lib.ptr(v_cache), int(k_cache.shape[0]), int(k_cache.shape[2]), _lib.ptr(out),
            _lib.stream_of(qkv),
        )
    return out


def tree_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    seqlen: torch.Tensor,
    parents: torch.Tensor,
    *,
    row_map: torch.Tensor | None = None,
    scale: float,
    window: int | None = None,
) -> torch.Tensor:
    """GQA attention of a tree's nodes: each over its row's sequence, its
    ancestors and itself (their K/V stored by ``apply_qkv_tree``), the last
    ``window`` of them with a window.  ``q [B, T, H, D]`` bf16; returns the same
    shape, 0 for padding.  ``seqlen[b]`` is node 0's position."""
    if q.ndim != 4 or q.dtype != torch.bfloat16:
        raise ValueError(f"tree_attention expects bf16 q [B, T, H, D], got {q.dtype} {tuple(q.shape)}.")
    bsz, nodes, n_q, head_dim = q.shape
    _check_rows("q", bsz, k_cache, v_cache, seqlen, row_map)
    n_kv, max_len = int(k_cache.shape[1]), int(k_cache.shape[2])
    _check_cache("tree_attention", k_cache, v_cache, n_kv, head_dim)
    if n_q % n_kv != 0:
        raise ValueError(f"n_q={n_q} not divisible by n_kv={n_kv}.")
    if window is not None and window < 1:
        raise ValueError(f"window must be positive, got {window}.")
    dev = q.device
    parents = _check_tree(parents, bsz, nodes, dev, "tree_attention")
    sl, rm = _i64(seqlen), _i64(row_map)
    _same_device("tree_attention", dev, k_cache, v_cache, sl, rm)
    q = q.contiguous()
    out = torch.empty_like(q)
    win = int(window or 0)
    nbytes = int(_lib.load().ma_tree_attn_workspace_bytes(bsz, nodes, n_q, n_kv, head_dim, max_len, win))
    with torch.cuda.device(dev):
        # scratch of this call alone: the allocator keeps it to this stream, a
        # captured graph to its own pool
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
        _lib.call(
            "ma_tree_attn",
            _lib.ptr(q), bsz, nodes, n_q, n_kv, head_dim, _lib.ptr(k_cache), _lib.ptr(v_cache),
            int(k_cache.shape[0]), max_len, _lib.ptr(sl), _lib.ptr(parents), _lib.ptr(rm), win, float(scale),
            _lib.ptr(out), _lib.ptr(ws), nbytes, _lib.stream_of(q),
        )
    return out


class TreeVerdict(NamedTuple):
    """``tokens [B, T]`` int64: the accepted tokens, the drawn one, then -1;
    ``accepted [B]`` int32: how many were accepted (-1: no sequence in the row);
    ``path [B, T]`` int32: the nodes from the root to the last accepted one, then
    -1."""

    tokens: torch.Tensor
    accepted: torch.Tensor
    path: torch.Tensor


def verify_tree(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    parents: torch.Tensor,
    uniform: torch.Tensor,
    *,
    temperature: float,
    top_p: float,
    top_k: int,
    draft_probs: torch.Tensor | None = None,
) -> TreeVerdict:
    """Accept drafted tokens against the target's law, then draw one more.

    The law at a node is ``fused_sample``'s (``top_k`` largest logits,
    temperature, nucleus ``top_p``; ``top_k=1`` is greedy).  From the root down,
    child ``c`` is accepted if ``uniform[b, c] * q(t) < P(t)``, else ``P`` becomes
    ``max(P - q, 0)`` normalised and the next child (in index order) is tried;
    ``uniform[b, 0]`` draws the last token.  ``draft_probs [B, T, V]``: row ``c``
    is the law that ``tokens[b, c]`` was drawn from (given its earlier siblings,
    where the draft draws without replacement); None: the tokens were chosen, not
    drawn.  The tokens returned follow the target's law.  ``logits [B, T, V]``,
    ``tokens [B, T]`` int64, ``uniform [B, T]`` float32 in [0, 1)."""
    if logits.ndim != 3:
        raise ValueError(f"verify_tree expects logits [B, T, vocab], got {tuple(logits.shape)}.")
    bsz, nodes, vocab = logits.shape
    _check(top_k, temperature, int(vocab))
    dev = logits.device
    parents = _check_tree(parents, bsz, nodes, dev, "verify_tree")
    if logits.stride(2) != 1 and vocab > 1:
        raise ValueError("logits rows must be contiguous.")
    if tokens.shape != (bsz, nodes) or uniform.shape != (bsz, nodes):
        raise ValueError(f"tokens {tuple(tokens.shape)} and uniform {tuple(uniform.shape)}, expected {(bsz, nodes)}.")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"tokens must be int64 or int32; got {tokens.dtype}.")
    if uniform.dtype != torch.float32:
        raise TypeError("uniform must be a float32 CUDA tensor.")
    tokens, uniform = tokens.to(torch.int64).contiguous(), uniform.contiguous()
    dt, p_dt, p_lb, p_lt = _lib.dtype_code(logits, "logits"), 0, 0, 0
    if draft_probs is not None:
        if draft_probs.shape != logits.shape:
            raise ValueError(f"draft_probs {tuple(draft_probs.shape)}, expected {tuple(logits.shape)}.")
        if draft_probs.stride(2) != 1 and vocab > 1:
            raise ValueError("draft_probs rows must be contiguous.")
        p_dt, p_lb, p_lt = _lib.dtype_code(draft_probs, "draft_probs"), draft_probs.stride(0), draft_probs.stride(1)
    _same_device("verify_tree", dev, tokens, uniform, draft_probs)
    out = TreeVerdict(torch.empty(bsz, nodes, device=dev, dtype=torch.int64),
                      torch.empty(bsz, device=dev, dtype=torch.int32),
                      torch.empty(bsz, nodes, device=dev, dtype=torch.int32))
    nbytes = int(_lib.load().ma_verify_tree_workspace_bytes(bsz, nodes, vocab, int(top_k)))
    with torch.cuda.device(dev):
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
        _lib.call(
            "ma_verify_tree",
            _lib.ptr(logits), dt, logits.stride(0), logits.stride(1), bsz, nodes, vocab, _lib.ptr(tokens),
            _lib.ptr(parents), _lib.ptr(uniform), _lib.ptr(draft_probs), p_dt, p_lb, p_lt, int(top_k),
            1.0 / float(temperature), float(top_p), _lib.ptr(ws), nbytes, _lib.ptr(out.tokens),
            _lib.ptr(out.accepted), _lib.ptr(out.path), _lib.stream_of(logits),
        )
    return out


def commit_tree(
    k_caches,
    v_caches,
    seqlen: torch.Tensor,
    path: torch.Tensor,
    accepted: torch.Tensor,
    *,
    row_map: torch.Tensor | None = None,
) -> torch.Tensor:
    """Move the accepted nodes' K/V of every layer (``k_caches`` / ``v_caches``:
    lists of caches) together behind each row's sequence; returns the new write
    positions ``seqlen + accepted + 1`` (int64 ``[B]``).  ``path`` / ``accepted``
    as ``verify_tree`` returns them."""
    if len(k_caches) == 0 or len(k_caches) != len(v_caches):
        raise ValueError(f"commit_tree expects as many K as V caches, got {len(k_caches)} and {len(v_caches)}.")
    if path.ndim != 2 or not 1 <= path.shape[1] <= MAX_NODES:
        raise ValueError(f"commit_tree expects path [B, T], T <= {MAX_NODES}, got {tuple(path.shape)}.")
    bsz, nodes = path.shape
    if accepted.shape != (bsz,):
        raise ValueError(f"accepted is {tuple(accepted.shape)}, expected {(bsz,)}.")
    if path.dtype != torch.int32 or accepted.dtype != torch.int32:
        raise TypeError("path and accepted must be int32.")
    first = k_caches[0]
    if first.ndim != 4:
        raise ValueError(f"commit_tree expects caches [rows, n_kv, max_len, head_dim], got {tuple(first.shape)}.")
    dev, shape = first.device, first.shape
    for t in (*k_caches, *v_caches):
        if t.shape != shape or t.dtype != torch.bfloat16 or not t.is_contiguous() or t.device != dev:
            raise ValueError("commit_tree: the caches must be contiguous bf16 tensors of one shape and device.")
    _check_rows("path", bsz, first, first, seqlen, row_map)
    sl, rm = _i64(seqlen), _i64(row_map)
    path, accepted = path.contiguous(), accepted.contiguous()
    _same_device("commit_tree", dev, sl, rm, path, accepted)
    out = torch.empty(bsz, device=dev, dtype=torch.int64)
    n = len(k_caches)
    kp = (ctypes.c_void_p * n)(*[t.data_ptr() for t in k_caches])
    vp = (ctypes.c_void_p * n)(*[t.data_ptr() for t in v_caches])
    with torch.cuda.device(dev):
        _lib.call("ma_tree_commit", kp, vp, n, bsz, nodes, int(shape[1]), int(shape[3]), int(shape[0]), int(shape[2]),
                  _lib.ptr(sl), _lib.ptr(path), _lib.ptr(accepted), _lib.ptr(rm), _lib.ptr(out),
                  _lib.stream_of(first))
    return out
