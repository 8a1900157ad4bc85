"""Decoding with a tree of drafted tokens per row.

A draft proposes, behind a row's last token, a tree of tokens; one pass of the
model scores them all and the branch that the target's law accepts is kept.  Per
layer ``apply_qkv_tree`` then ``tree_attention``, on the logits ``verify_tree``,
and ``commit_tree`` on the cache (``decode_graph.tree_step`` runs them).  No
reference counterpart: its decode step takes one token per row
(``src/maple_run/kernels/decode_attn.py:362-592``, whose QK-norm, RoPE, K/V
store and GQA these are for several, and ``src/maple_run/kernels/sampler.py``,
whose law the verification keeps).

The tree is ``parents [B, T]``, ``T <= 64``, on the device: node 0 is the row's
last token (its K/V not yet cached) with parent -1, any other node's parent comes
before it (``0 <= parents[b, i] < i``).  A node with any other parent, and all
below it, is padding; a row whose entry 0 is not -1 has no sequence.  Node ``i``
is cached at ``seqlen[b] + i`` and stands at position ``seqlen[b] + depth``.
Nodes past the cache's end are neither stored nor attended, so they must not be
accepted either: where ``seqlen[b] + T`` may exceed ``max_len``, all four get the
tree from ``fit_tree``, in which such nodes are padding.  ``row_map`` (slot ->
cache row) names each cache row once.
"""

from __future__ import annotations

import array
from operator import attrgetter
from typing import NamedTuple

import torch

from .. import _lib
from .sampler import _check

MAX_NODES = 64
_FAR = 2 ** 62

# Decoding calls these once per layer and step, so the checks below read each
# property once and nothing goes through a context manager or a stream object
# that a call does not need.  (None in a torch built without GPU support, whose
# tensors no call gets past _device with.)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current = getattr(torch._C, "_cuda_getDevice", None)


def _call(idx: int, name: str, *args) -> None:
    """``name`` with the tensors' device current, on its current stream."""
    if _current() == idx:
        _lib.call(name, *args, _stream(idx))
    else:
        with torch.cuda.device(idx):
            _lib.call(name, *args, _stream(idx))


_index = torch.Tensor.get_device


def _device(what: str, *tensors: torch.Tensor) -> int:
    """The one device that all of the tensors are on."""
    idx = tensors[0].get_device()
    if idx < 0:
        raise RuntimeError(f"{what} requires CUDA tensors.")
    if set(map(_index, tensors)) != {idx}:
        raise ValueError(f"{what}: tensors on several devices: {[str(t.device) for t in tensors]}.")
    return idx


def _check_parents(what: str, parents: torch.Tensor, bsz: int, nodes: int) -> None:
    if not 1 <= nodes <= MAX_NODES:
        raise ValueError(f"{what}: a tree has 1 to {MAX_NODES} nodes, got {nodes}.")
    if parents.shape != (bsz, nodes):
        raise ValueError(f"{what}: parents is {tuple(parents.shape)}, expected {(bsz, nodes)}.")
    if parents.dtype != torch.int32 and parents.dtype != torch.int64:
        raise TypeError(f"{what}: parents must be int32 or int64; got {parents.dtype}.")


def check_tree(what: str, parents: torch.Tensor, bsz: int, nodes: int) -> torch.Tensor:
    """``parents`` as the kernels take them: int32 ``[bsz, nodes]``, contiguous."""
    _check_parents(what, parents, bsz, nodes)
    if parents.dtype != torch.int32:
        parents = parents.clamp(-2, MAX_NODES).to(torch.int32)  # (no large value may wrap to a node)
    return parents if parents.is_contiguous() else parents.contiguous()


def _positions(name: str, t: torch.Tensor, bsz: int) -> torch.Tensor:
    if t.numel() != bsz:
        raise ValueError(f"{name} has {t.numel()} entries, expected {bsz}.")
    if t.dtype != torch.int64:
        if t.dtype.is_floating_point or t.dtype == torch.bool:
            raise TypeError(f"{name} must hold whole numbers; got {t.dtype}.")
        t = t.to(torch.int64)
    return t if t.is_contiguous() else t.contiguous()


def fit_tree(parents: torch.Tensor, seqlen: torch.Tensor, max_len: int) -> torch.Tensor:
    """``parents`` (int32) without the nodes that a cache of ``max_len`` positions
    has no place for: node ``i`` of row ``b`` is padding where ``seqlen[b] + i >=
    max_len``, and a full row has no sequence.  A node's slot lies behind its
    parent's, so whatever is kept is kept with its branch, and an accepted branch
    ends within the cache.  Capturable."""
    if parents.ndim != 2:
        raise ValueError(f"fit_tree expects parents [B, T], got {tuple(parents.shape)}.")
    bsz, nodes = parents.shape
    _check_parents("fit_tree", parents, bsz, nodes)
    sl = _positions("seqlen", seqlen, bsz)
    parents = parents.contiguous()
    idx = _device("fit_tree", parents, sl)
    out = torch.empty_like(parents, dtype=torch.int32)
    _call(idx, "ma_tree_fit", parents.data_ptr(), int(parents.dtype == torch.int64), bsz, nodes, sl.data_ptr(),
          max_len, out.data_ptr())
    return out


def _cache(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor, bsz: int, row_map: torch.Tensor | None):
    """The caches' shape ``[rows, n_kv, max_len, head_dim]``."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"{what}: K {tuple(shape)} and V {tuple(v_cache.shape)} caches, "
                         "expected [rows, n_kv, max_len, head_dim] twice.")
    if k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        raise TypeError("the KV cache must be bf16.")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("the KV cache must be contiguous [rows, n_kv, max_len, head_dim].")
    if row_map is None and shape[0] != bsz:
        raise ValueError(f"KV cache batch {shape[0]} != {what} batch {bsz}.")
    return shape


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
    ldb, ldt, one = qkv.stride()
    if one != 1:
        raise ValueError("apply_qkv_tree needs a row-contiguous qkv.")
    rows, n_kv, max_len, d = _cache("apply_qkv_tree", k_cache, v_cache, bsz, row_map)
    if n_kv != num_kv_heads or d != head_dim:
        raise ValueError(f"apply_qkv_tree: cache {tuple(k_cache.shape)} for {num_kv_heads} KV heads of {head_dim}.")
    more, qw, kw, c, s = [], None, None, None, None
    w_dt = dt = ld = n_pos = mode = 0
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
    if use_rope and rotary_dim != 0:
        mode, shape, strides = 2 if interleaved else 1, cos_table.shape, cos_table.stride()
        if (len(shape) != 2 or sin_table.shape != shape or sin_table.stride() != strides or strides[1] != 1
                or sin_table.dtype != cos_table.dtype):
            raise ValueError("cos and sin tables must share dtype and layout, rows contiguous.")
        n_pos, ld = shape[0], strides[0]
        if n_pos < 1 or shape[1] < rotary_dim:
            raise ValueError(f"tables {tuple(shape)} for a rotary_dim of {rotary_dim}.")
        dt = _lib.dtype_code(cos_table, "cos_table")
        more += [cos_table, sin_table]
        c, s = cos_table.data_ptr(), sin_table.data_ptr()
    parents = check_tree("apply_qkv_tree", parents, bsz, nodes)
    sl = _positions("seqlen", seqlen, bsz)
    rm = None
    if row_map is not None:
        more.append(_positions("row_map", row_map, bsz))
        rm = more[-1].data_ptr()
    idx = _device("apply_qkv_tree", qkv, k_cache, v_cache, sl, parents, *more)
    out = qkv.new_empty((bsz, nodes, num_heads, head_dim))
    _call(
        idx, "ma_tree_qkv",
        qkv.data_ptr(), ldb, ldt, bsz, nodes, num_heads, num_kv_heads, head_dim, qw, kw, w_dt,
        c, s, dt, ld, n_pos, rotary_dim if mode else 0, mode, eps, sl.data_ptr(),
        parents.data_ptr(), rm, k_cache.data_ptr(), v_cache.data_ptr(), rows, max_len, out.data_ptr(),
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
    rows, n_kv, max_len, d = _cache("tree_attention", k_cache, v_cache, bsz, row_map)
    if d != head_dim:
        raise ValueError(f"tree_attention: cache {tuple(k_cache.shape)} for heads of {head_dim}.")
    if n_kv < 1 or n_q % n_kv != 0:
        raise ValueError(f"n_q={n_q} not divisible by n_kv={n_kv}.")
    if window is None:
        window = 0
    elif window < 1:
        raise ValueError(f"window must be positive, got {window}.")
    elif window > _FAR:
        window = _FAR  # (past every position; more would wrap in 64 bits)
    parents = check_tree("tree_attention", parents, bsz, nodes)
    sl = _positions("seqlen", seqlen, bsz)
    rm = None if row_map is None else _positions("row_map", row_map, bsz)
    idx = _device("tree_attention", q, k_cache, v_cache, sl, parents, *(() if rm is None else (rm,)))
    q = q.contiguous()
    out = torch.empty_like(q)
    nbytes = _lib.load().ma_tree_attn_workspace_bytes(bsz, nodes, n_q, n_kv, head_dim, max_len, window)
    # scratch of this call alone: the allocator keeps it to this stream, a
    # captured graph to its own pool
    ws = q.new_empty(nbytes // 2) if nbytes else None
    _call(
        idx, "ma_tree_attn",
        q.data_ptr(), bsz, nodes, n_q, n_kv, head_dim, k_cache.data_ptr(), v_cache.data_ptr(), rows, max_len,
        sl.data_ptr(), parents.data_ptr(), _lib.ptr(rm), window, scale, out.data_ptr(), _lib.ptr(ws), nbytes,
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
    shape = logits.shape
    bsz, nodes, vocab = shape
    _check(top_k, temperature, vocab)
    l_dt = _lib.dtype_code(logits, "logits")
    parents = check_tree("verify_tree", parents, bsz, nodes)
    ldb, ldt, one = logits.stride()
    if one != 1 and vocab > 1:
        raise ValueError("logits rows must be contiguous.")
    if tokens.shape != (bsz, nodes) or uniform.shape != (bsz, nodes):
        raise ValueError(f"tokens {tuple(tokens.shape)} and uniform {tuple(uniform.shape)}, expected {(bsz, nodes)}.")
    if tokens.dtype != torch.int64:
        if tokens.dtype != torch.int32:
            raise TypeError(f"tokens must be int64 or int32; got {tokens.dtype}.")
        tokens = tokens.to(torch.int64)
    if uniform.dtype != torch.float32:
        raise TypeError("uniform must be a float32 CUDA tensor.")
    tokens, uniform = tokens.contiguous(), uniform.contiguous()
    p_dt = p_lb = p_lt = 0
    if draft_probs is not None:
        if draft_probs.shape != shape:
            raise ValueError(f"draft_probs {tuple(draft_probs.shape)}, expected {tuple(shape)}.")
        p_lb, p_lt, one = draft_probs.stride()
        if one != 1 and vocab > 1:
            raise ValueError("draft_probs rows must be contiguous.")
        p_dt = _lib.dtype_code(draft_probs, "draft_probs")
    idx = _device("verify_tree", logits, tokens, parents, uniform, *(() if draft_probs is None else (draft_probs,)))
    out = TreeVerdict(torch.empty_like(tokens), parents.new_empty(bsz), torch.empty_like(parents))
    nbytes = _lib.load().ma_verify_tree_workspace_bytes(bsz, nodes, vocab, top_k)
    ws = tokens.new_empty(nbytes // 8)  # scratch of this call alone, as in tree_attention
    _call(
        idx, "ma_verify_tree",
        logits.data_ptr(), l_dt, ldb, ldt, bsz, nodes, vocab, tokens.data_ptr(),
        parents.data_ptr(), uniform.data_ptr(), _lib.ptr(draft_probs), p_dt, p_lb, p_lt, top_k,
        1.0 / float(temperature), top_p, ws.data_ptr(), nbytes, out[0].data_ptr(), out[1].data_ptr(),
        out[2].data_ptr(),
    )
    return out


_shape, _dtype = attrgetter("shape"), attrgetter("dtype")


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
    as ``verify_tree`` returns them for a tree that fits the cache (``fit_tree``):
    a node that was never stored has no K/V to move."""
    n = len(k_caches)
    if n == 0 or n != len(v_caches):
        raise ValueError(f"commit_tree expects as many K as V caches, got {n} and {len(v_caches)}.")
    if path.ndim != 2 or not 1 <= path.shape[1] <= MAX_NODES:
        raise ValueError(f"commit_tree expects path [B, T], T <= {MAX_NODES}, got {tuple(path.shape)}.")
    bsz, nodes = path.shape
    if accepted.shape != (bsz,):
        raise ValueError(f"accepted is {tuple(accepted.shape)}, expected {(bsz,)}.")
    if path.dtype != torch.int32 or accepted.dtype != torch.int32:
        raise TypeError("path and accepted must be int32.")
    caches = [*k_caches, *v_caches]
    first = caches[0]
    shape = _cache("commit_tree", first, caches[n], bsz, row_map)
    # every layer's cache like the first (a set each: one pass without bytecode)
    if (set(map(_shape, caches)) != {shape} or set(map(_dtype, caches)) != {torch.bfloat16}
            or not all(map(torch.Tensor.is_contiguous, caches))):
        raise ValueError("commit_tree: the caches must be contiguous bf16 tensors of one shape.")
    ptrs = array.array("Q", map(torch.Tensor.data_ptr, caches))
    if len(set(ptrs)) != 2 * n:
        raise ValueError("commit_tree: the same cache twice.")
    sl = _positions("seqlen", seqlen, bsz)
    rm = None if row_map is None else _positions("row_map", row_map, bsz)
    path, accepted = path.contiguous(), accepted.contiguous()
    idx = _device("commit_tree", *caches, sl, path, accepted, *(() if rm is None else (rm,)))
    out = sl.new_empty(bsz)
    at = ptrs.buffer_info()[0]
    _call(
        idx, "ma_tree_commit",
        at, at + 8 * n, n, bsz, nodes, shape[1], shape[3], shape[0], shape[2], sl.data_ptr(), path.data_ptr(),
        accepted.data_ptr(), _lib.ptr(rm), out.data_ptr(),
    )
    return out
