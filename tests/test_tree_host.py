"""Host side of decoding with drafted trees (CPU): refusals of the C entry points
and of the wrappers before any launch, and the workspace queries."""

from __future__ import annotations

import pytest
import torch

from maple_amd import _lib, kernels
from maple_amd.decode_graph import Sampling, tree_step
from maple_amd.kernels import tree

FAKE = 0x10000  # a pointer that is never dereferenced: the call is refused before its launch


def qkv_args(**kw):
    a = dict(qkv=FAKE, ldb=1024, ldt=512, batch=1, nodes=2, h=4, hkv=2, d=64, qw=FAKE, kw=FAKE, w_dt=0, cos=FAKE,
             sin=FAKE, cs_dt=0, ld_cs=32, n_pos=64, rot=32, mode=1, eps=1e-6, seqlen=FAKE, parents=FAKE, row_map=None,
             k=FAKE, v=FAKE, rows=1, max_len=64, out=FAKE, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,match", [
    (dict(nodes=0), "1 to 64 nodes"), (dict(nodes=65), "1 to 64 nodes"), (dict(d=96), "head_dim"),
    (dict(h=5), "query heads"), (dict(hkv=0), "query heads"), (dict(h=65536, hkv=1), "query heads"), (dict(batch=2), "cache sizes"),
    (dict(batch=70000, rows=70000), "too large"), (dict(rot=31), "rotary_dim"), (dict(rot=66), "rotary_dim"),
    (dict(mode=3), "rotary_dim"), (dict(cos=None), "tables"), (dict(n_pos=0), "tables"), (dict(ld_cs=16), "tables"),
    (dict(qw=None), "norm weight"), (dict(qkv=None), "null"), (dict(parents=None), "null"),
    (dict(k=FAKE + 2), "aligned"), (dict(out=FAKE + 8), "aligned")])
def test_tree_qkv_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _lib.call("ma_tree_qkv", *qkv_args(**kw))


def attn_args(**kw):
    a = dict(q=FAKE, batch=1, nodes=2, h=4, hkv=2, d=64, k=FAKE, v=FAKE, rows=1, max_len=4096, seqlen=FAKE,
             parents=FAKE, row_map=None, window=0, scale=0.125, out=FAKE, ws=FAKE, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,match", [
    (dict(nodes=65), "1 to 64 nodes"), (dict(d=32), "head_dim"), (dict(h=3), "query heads"), (dict(window=-1), "window"),
    (dict(seqlen=None), "null"), (dict(q=FAKE + 4), "aligned"), (dict(ws=FAKE + 4), "aligned"),
    (dict(ws=None), "workspace"), (dict(ws_bytes=8), "workspace"), (dict(max_len=0), "cache sizes"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale")])
def test_tree_attn_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _lib.call("ma_tree_attn", *attn_args(**kw))


def verify_args(**kw):
    a = dict(logits=FAKE, dt=1, ldb=100, ldt=50, batch=1, nodes=2, vocab=50, tokens=FAKE, parents=FAKE, uniform=FAKE,
             probs=None, p_dt=0, p_ldb=0, p_ldt=0, top_k=5, inv_t=1.0, top_p=1.0, ws=FAKE, ws_bytes=1 << 40, out=FAKE,
             accepted=FAKE, path=FAKE, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,match", [
    (dict(nodes=0), "1 to 64 nodes"), (dict(nodes=65), "1 to 64 nodes"), (dict(vocab=0), "vocabulary"),
    (dict(vocab=1 << 32), "vocabulary"), (dict(top_k=0), "top_k"), (dict(top_k=65, vocab=100), "top_k"),
    (dict(top_k=51), "top_k"), (dict(inv_t=0.0), "temperature"), (dict(inv_t=float("inf")), "temperature"),
    (dict(top_p=0.0), "top_p"), (dict(top_p=1.5), "top_p"), (dict(logits=None), "null"), (dict(logits=FAKE + 1), "aligned"),
    (dict(ws_bytes=0), "workspace"), (dict(ws=None), "workspace"), (dict(batch=40000), "too large")])
def test_verify_tree_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _lib.call("ma_verify_tree", *verify_args(**kw))


@pytest.mark.parametrize("kw", [dict(dt=7), dict(probs=FAKE, p_dt=7)])
def test_verify_tree_refuses_types(kw):
    with pytest.raises(TypeError):
        _lib.call("ma_verify_tree", *verify_args(**kw))


def test_tree_commit_refuses():
    import ctypes

    ok = (ctypes.c_void_p * 2)(FAKE, FAKE + 64)
    bad = (ctypes.c_void_p * 2)(FAKE, FAKE + 8)
    null = (ctypes.c_void_p * 2)(FAKE, None)

    def call(k=ok, v=ok, layers=2, batch=1, nodes=4, hkv=2, d=64, rows=1, max_len=64, seqlen=FAKE, path=FAKE,
             accepted=FAKE, new=FAKE + 8):
        _lib.call("ma_tree_commit", k, v, layers, batch, nodes, hkv, d, rows, max_len, seqlen, path, accepted, None,
                  new, None)

    for kw, match in ((dict(nodes=65), "nodes"), (dict(d=80), "head_dim"), (dict(layers=0), "sizes"),
                      (dict(batch=2), "cache sizes"), (dict(v=bad), "aligned"), (dict(k=null), "null"),
                      (dict(path=None), "null"), (dict(new=FAKE), "new_seqlen")):
        with pytest.raises(ValueError, match=match):
            call(**kw)


def test_empty_batches_are_no_work():
    for name, args in (("ma_tree_qkv", qkv_args(batch=0, rows=0)), ("ma_tree_attn", attn_args(batch=0, rows=0)),
                       ("ma_verify_tree", verify_args(batch=0, ws=None, ws_bytes=0))):
        _lib.call(name, *args)


def test_workspace_queries():
    lib = _lib.load()
    assert lib.ma_tree_attn_workspace_bytes(1, 8, 32, 4, 64, 4224, 0) > 0
    assert lib.ma_tree_attn_workspace_bytes(1, 8, 32, 4, 64, 32, 0) == 0  # one split: no sums to keep
    assert lib.ma_tree_attn_workspace_bytes(1, 65, 32, 4, 64, 4224, 0) == 0
    assert lib.ma_verify_tree_workspace_bytes(1, 1, 50, 5) == 5 * 8  # one segment: its keys alone
    assert lib.ma_verify_tree_workspace_bytes(1, 8, 151936, 1) > 8 * 8
    # a short window needs no more splits than it has positions
    assert (lib.ma_tree_attn_workspace_bytes(1, 8, 32, 4, 64, 1 << 20, 512)
            < lib.ma_tree_attn_workspace_bytes(1, 8, 32, 4, 64, 1 << 20, 0))


def _cpu(**kw):
    b, t = 2, 3
    a = dict(qkv=torch.zeros(b, t, 8 * 64, dtype=torch.bfloat16), w=torch.ones(64), cos=torch.ones(8, 32),
             k=torch.zeros(b, 2, 8, 64, dtype=torch.bfloat16), seqlen=torch.zeros(b, dtype=torch.int64),
             parents=torch.full((b, t), -1, dtype=torch.int32))
    a.update(kw)
    return a


def _qkv(a, **kw):
    kw = {**dict(num_heads=4, num_kv_heads=2, head_dim=64, rotary_dim=32), **kw}
    return kernels.apply_qkv_tree(a["qkv"], a["w"], a.get("w2", a["w"]), a["cos"], a.get("sin", a["cos"]), a["k"],
                                  a.get("v", a["k"]), a["seqlen"], a["parents"], row_map=a.get("row_map"), **kw)


def test_apply_qkv_tree_checks_its_arguments():
    with pytest.raises(RuntimeError, match="CUDA"):
        _qkv(_cpu())
    for kw, err in ((dict(qkv=torch.zeros(2, 3, 512)), ValueError),
                    (dict(qkv=torch.zeros(2, 512, 3, dtype=torch.bfloat16).transpose(1, 2)), ValueError),
                    (dict(qkv=torch.zeros(2, 3, 513, dtype=torch.bfloat16)), ValueError),
                    (dict(k=torch.zeros(3, 2, 8, 64, dtype=torch.bfloat16)), ValueError),
                    (dict(k=torch.zeros(2, 4, 8, 64, dtype=torch.bfloat16)), ValueError),
                    (dict(k=torch.zeros(2, 2, 8, 64)), TypeError),
                    (dict(v=torch.zeros(2, 2, 9, 64, dtype=torch.bfloat16)), ValueError),
                    (dict(seqlen=torch.zeros(3, dtype=torch.int64)), ValueError),
                    (dict(seqlen=torch.zeros(2)), TypeError),
                    (dict(parents=torch.zeros(2, 4, dtype=torch.int32)), ValueError),
                    (dict(parents=torch.zeros(2, 3)), TypeError),
                    (dict(w2=torch.ones(64, dtype=torch.bfloat16)), TypeError),
                    (dict(w=torch.ones(32)), ValueError), (dict(w2=None), ValueError),
                    (dict(cos=torch.ones(8, 16)), ValueError), (dict(sin=torch.ones(9, 32)), ValueError),
                    (dict(cos=torch.ones(8, 32, dtype=torch.float64)), TypeError),
                    (dict(row_map=torch.zeros(1, dtype=torch.int64)), ValueError)):
        with pytest.raises(err):
            _qkv(_cpu(**kw))


def test_tree_attention_checks_its_arguments():
    a = _cpu()

    def call(q=torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16), **kw):
        args = {**dict(scale=0.125), **kw}
        return tree.tree_attention(q, a["k"], a["k"], a["seqlen"], args.pop("parents", a["parents"]), **args)

    with pytest.raises(RuntimeError, match="CUDA"):
        call()
    for q, kw in ((torch.zeros(2, 3, 4, 64), {}), (torch.zeros(2, 3, 4, 128, dtype=torch.bfloat16), {}),
                  (torch.zeros(2, 3, 3, 64, dtype=torch.bfloat16), {}), (torch.zeros(2, 3, 64, dtype=torch.bfloat16), {}),
                  (torch.zeros(2, 70, 4, 64, dtype=torch.bfloat16), dict(parents=torch.zeros(2, 70, dtype=torch.int32)))):
        with pytest.raises(ValueError):
            call(q, **kw)
    for w in (0, -3):
        with pytest.raises(ValueError, match="window"):
            call(window=w)


def test_verify_tree_checks_its_arguments():
    def call(logits=torch.zeros(2, 3, 50), tokens=torch.zeros(2, 3, dtype=torch.int64),
             parents=torch.full((2, 3), -1, dtype=torch.int32), uniform=torch.zeros(2, 3), **kw):
        return kernels.verify_tree(logits, tokens, parents, uniform,
                                   **{**dict(temperature=1.0, top_p=1.0, top_k=5), **kw})

    with pytest.raises(RuntimeError, match="CUDA"):
        call()
    for kw, err in ((dict(logits=torch.zeros(6, 50)), ValueError), (dict(logits=torch.zeros(2, 3, 50, dtype=torch.int32)), TypeError),
                    (dict(logits=torch.zeros(2, 50, 3).transpose(1, 2)), ValueError), (dict(top_k=0), ValueError),
                    (dict(top_k=65, logits=torch.zeros(2, 3, 100)), ValueError), (dict(top_k=51), ValueError),
                    (dict(temperature=0.0), ValueError), (dict(tokens=torch.zeros(2, 3)), TypeError),
                    (dict(tokens=torch.zeros(2, 2, dtype=torch.int64)), ValueError),
                    (dict(uniform=torch.zeros(2, 3, dtype=torch.float64)), TypeError),
                    (dict(uniform=torch.zeros(6)), ValueError), (dict(draft_probs=torch.zeros(2, 3, 49)), ValueError),
                    (dict(draft_probs=torch.zeros(2, 3, 50, dtype=torch.float64)), TypeError)):
        with pytest.raises(err):
            call(**kw)


def test_commit_tree_checks_its_arguments():
    k = [torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16) for _ in range(4)]

    def call(ks=tuple(k[:2]), vs=tuple(k[2:]), seqlen=torch.zeros(2, dtype=torch.int64),
             path=torch.zeros(2, 3, dtype=torch.int32), accepted=torch.zeros(2, dtype=torch.int32)):
        return kernels.commit_tree(list(ks), list(vs), seqlen, path, accepted)

    with pytest.raises(RuntimeError, match="CUDA"):
        call()
    for kw, err in ((dict(ks=()), ValueError), (dict(ks=k[:1]), ValueError), (dict(vs=(k[0], k[3])), ValueError),
                    (dict(vs=(k[2], torch.zeros(2, 2, 9, 64, dtype=torch.bfloat16))), ValueError),
                    (dict(vs=(k[2], torch.zeros(2, 2, 8, 64))), ValueError),
                    (dict(path=torch.zeros(2, 3, dtype=torch.int64)), TypeError),
                    (dict(accepted=torch.zeros(3, dtype=torch.int32)), ValueError),
                    (dict(path=torch.zeros(2, 65, dtype=torch.int32)), ValueError),
                    (dict(seqlen=torch.zeros(1, dtype=torch.int64)), ValueError)):
        with pytest.raises(err):
            call(**kw)


def test_tree_step_refuses_settings_the_sampler_does_not_cover():
    with pytest.raises(ValueError, match="sampling"):
        tree_step(None, None, torch.zeros(1, 1, dtype=torch.int64), torch.full((1, 1), -1, dtype=torch.int32),
                  Sampling(temperature=1.0, top_k=0))


def test_fit_tree_checks_its_arguments():
    parents, seqlen = torch.full((2, 3), -1), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.fit_tree(parents, seqlen, 8)
    for args, err in (((parents, seqlen[:1], 8), ValueError), ((parents.float(), seqlen, 8), TypeError),
                      ((parents, seqlen.float(), 8), TypeError), ((parents[0], seqlen, 8), ValueError),
                      ((torch.zeros(2, 65, dtype=torch.int32), seqlen, 8), ValueError)):
        with pytest.raises(err):
            kernels.fit_tree(*args)
    for kw, match in ((dict(nodes=65), "1 to 64 nodes"), (dict(nodes=0), "1 to 64 nodes"), (dict(batch=40000), "too large"),
                      (dict(max_len=-1), "cache sizes"), (dict(parents=None), "null"), (dict(out=None), "null")):
        a = {**dict(parents=FAKE, wide=0, batch=1, nodes=2, seqlen=FAKE, max_len=8, out=FAKE, stream=None), **kw}
        with pytest.raises(ValueError, match=match):
            _lib.call("ma_tree_fit", *a.values())
    _lib.call("ma_tree_fit", FAKE, 0, 0, 2, FAKE, 8, FAKE, None)  # an empty batch is no work


class _Stub:
    """What ``forward_tree`` needs of a decoder and a cache; notes the trees that its layers get."""

    def __init__(self, layers=3):
        import types

        self.cfg, self.flash_head, self.trees = types.SimpleNamespace(layers=layers), None, []

    def slot_rows(self, width):
        return torch.zeros(width, dtype=torch.int64), None

    def embed_tokens(self, ids):
        return torch.zeros(ids.numel(), 4)

    def _layer(self, i, hidden, cache, routing, qkv, tree):
        self.trees.append(tree)
        return hidden, None

    def head(self, hidden, *_):
        return torch.zeros(hidden.shape[0], 7)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_forward_tree_converts_its_tree_once(dtype):
    from maple_amd.model import SyntheticDecoder

    stub, parents = _Stub(), torch.tensor([[-1, 0, 0], [-1, 0, -1]], dtype=dtype)
    out = SyntheticDecoder.forward_tree(stub, torch.zeros(2, 3, dtype=torch.int64), parents, stub)
    assert out.shape == (2, 3, 7) and len(stub.trees) == 3
    for tree_ in stub.trees:
        assert tree_ is stub.trees[0] and tree_.dtype == torch.int32 and tree_.tolist() == parents.tolist()


@pytest.mark.parametrize("shape", [(3, 2), (2, 4), (1, 6), (6,), (3, 3)])
def test_forward_tree_refuses_parents_of_another_shape(shape):
    from maple_amd.model import SyntheticDecoder

    stub = _Stub()
    with pytest.raises(ValueError):
        SyntheticDecoder.forward_tree(stub, torch.zeros(2, 3, dtype=torch.int64),
                                      torch.full(shape, -1, dtype=torch.int32), stub)
    assert not stub.trees


def test_the_package_imports_with_a_torch_without_gpu_support():
    import subprocess
    import sys
    from pathlib import Path

    code = ("import torch\n"
            "for n in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n"
            "    if hasattr(torch._C, n): delattr(torch._C, n)\n"
            "import __graft_entry__\n"
            "__graft_entry__.load_package()\n"
            "import maple_amd.kernels, maple_amd.model, maple_amd.decode_graph\n"
            "a = dict(dtype=torch.bfloat16)\n"
            "try:\n"
            "    maple_amd.kernels.tree_attention(torch.zeros(1, 1, 1, 64, **a), torch.zeros(1, 1, 4, 64, **a),\n"
            "        torch.zeros(1, 1, 4, 64, **a), torch.zeros(1, dtype=torch.int64),\n"
            "        torch.full((1, 1), -1, dtype=torch.int32), scale=1.0)\n"
            "except RuntimeError as e:\n"
            "    print('refused:', e)\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], timeout=300,
                          stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    assert done.returncode == 0, done.stderr
    assert "refused: tree_attention requires CUDA tensors" in done.stdout


def test_windows_past_64_bits_are_none(monkeypatch):
    """A window larger than any position sees everything; it does not wrap."""
    a, windows = _cpu(), []
    monkeypatch.setattr(tree, "_device", lambda what, *t: 0)
    monkeypatch.setattr(tree, "_call", lambda idx, name, *args: windows.append(args[13]))
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    for window in (None, 1, 512, 2 ** 63 - 1, 2 ** 63, 2 ** 64, 2 ** 64 + 5, 2 ** 200):
        tree.tree_attention(q, a["k"], a["k"], a["seqlen"], a["parents"], scale=0.125, window=window)
    assert windows[:3] == [0, 1, 512] and all(w == 0 or 2 ** 62 <= w < 2 ** 63 for w in windows[3:])


@pytest.mark.parametrize("scale", [3e38, -3e38])
def test_tree_attn_refuses_scales_that_overflow(scale):
    """The scores are taken in powers of two: scale x log2 e has to be a float32 value."""
    with pytest.raises(ValueError, match="scale"):
        _lib.call("ma_tree_attn", *attn_args(scale=scale, batch=0, rows=0))
    _lib.call("ma_tree_attn", *attn_args(scale=scale / 2, batch=0, rows=0))
