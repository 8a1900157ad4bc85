"""What the quantised cache's and the shared prefixes' calls refuse (no GPU: the
checks run before anything is launched)."""

from __future__ import annotations

import pytest
import torch

from maple_amd import _lib
from maple_amd.kernels import (KV, QuantKV, SharedPrefix, apply_qkv_quant, dequantize_kv, make_quant_kv,
                               prefix_gqa_attn, quant_attention, quant_gqa_attn, quantize_kv)

BF = torch.bfloat16
FAKE = 0x10000


def cache(rows=2, nkv=2, n=16, d=64):
    return make_quant_kv(rows, nkv, n, d, "cpu")


def plain(rows=2, nkv=2, n=16, d=64):
    return KV(torch.zeros(rows, nkv, n, d, dtype=BF), torch.zeros(rows, nkv, n, d, dtype=BF))


def n64(*x):
    return torch.tensor(x, dtype=torch.int64)


def test_an_empty_cache_holds_zeros():
    c = cache()
    assert c.k.dtype == torch.float8_e4m3fn and c.k_scale.dtype == torch.float8_e8m0fnu
    assert (c.k.float() == 0).all() and torch.isfinite(c.v_scale.float()).all()
    assert sum(t.numel() for t in c) == 2 * 2 * 2 * 16 * (64 + 1)


QKV = dict(num_heads=4, num_kv_heads=2, head_dim=64, rotary_dim=32)


def qkv_call(of=apply_qkv_quant, **kw):
    a = dict(qkv=torch.zeros(2, 8 * 64, dtype=BF), q_weight=torch.ones(64), k_weight=torch.ones(64),
             cos_table=torch.zeros(16, 32), sin_table=torch.zeros(16, 32), cache=cache(), seqlen=n64(0, 1), **QKV)
    a.update(kw)
    return of(**a)


QKV_REFUSED = [
    (dict(), RuntimeError, "CUDA"),
    (dict(cache=plain()), TypeError, "QuantKV"),
    (dict(qkv=torch.zeros(2, 8 * 64)), ValueError, "bf16"),
    (dict(qkv=torch.zeros(2, 1, 8 * 64, dtype=BF)), ValueError, "bf16"),
    (dict(qkv=torch.zeros(2, 7 * 64, dtype=BF)), ValueError, "rows of"),
    (dict(qkv=torch.zeros(8 * 64, 2, dtype=BF).t()), ValueError, "row-contiguous"),
    (dict(cache=cache(rows=3)), ValueError, "batch"),
    (dict(cache=cache(nkv=1)), ValueError, "KV heads"),
    (dict(cache=cache(d=128)), ValueError, "KV heads"),
    (dict(cache=QuantKV(*cache()[:3], cache(n=15).v_scale)), ValueError, "scales"),
    (dict(cache=QuantKV(*cache()[:3], torch.zeros(2, 2, 16))), TypeError, "scales"),
    (dict(cache=QuantKV(*plain(), *cache()[2:])), TypeError, "caches"),
    (dict(cache=QuantKV(*(t.transpose(0, 1) for t in cache()))), ValueError, "contiguous"),
    (dict(q_weight=None), ValueError, "together"),
    (dict(q_weight=torch.ones(64, dtype=BF)), TypeError, "dtype"),
    (dict(q_weight=torch.ones(32), k_weight=torch.ones(32)), ValueError, "entries"),
    (dict(q_weight=torch.ones(64, dtype=torch.float64), k_weight=torch.ones(64, dtype=torch.float64)), TypeError, "q_weight"),
    (dict(cos_table=torch.zeros(16, 30)), ValueError, "tables"),
    (dict(cos_table=torch.zeros(16, 30), sin_table=torch.zeros(16, 30)), ValueError, "rotary_dim"),
    (dict(cos_table=torch.zeros(0, 32), sin_table=torch.zeros(0, 32)), ValueError, "rotary_dim"),
    (dict(seqlen=n64(0)), ValueError, "seqlen"),
    (dict(seqlen=torch.zeros(2)), TypeError, "whole"),
    (dict(positions=n64(0, 1, 2)), ValueError, "positions"),
    (dict(row_map=torch.ones(2)), TypeError, "row_map"),
]


@pytest.mark.parametrize("kw,error,match", QKV_REFUSED)
def test_qkv_refuses(kw, error, match):
    with pytest.raises(error, match=match):
        qkv_call(**kw)


@pytest.mark.parametrize("kw,error,match", QKV_REFUSED + [(dict(window=0), ValueError, "window"),
                                                         (dict(window=-1), ValueError, "window")])
def test_fused_attention_refuses(kw, error, match):
    with pytest.raises(error, match=match):
        qkv_call(quant_attention, scale=0.125, **kw)


@pytest.mark.parametrize("kw,error,match", [
    (dict(), RuntimeError, "CUDA"),
    (dict(cache=plain()), TypeError, "QuantKV"),
    (dict(k=torch.zeros(2, 2, 5, 64)), TypeError, "bf16"),
    (dict(v=torch.zeros(2, 2, 4, 64, dtype=BF)), ValueError, "k and v"),
    (dict(k=torch.zeros(2, 5, 64, dtype=BF), v=torch.zeros(2, 5, 64, dtype=BF)), ValueError, "k and v"),
    (dict(k=torch.zeros(2, 2, 64, 5, dtype=BF).transpose(2, 3)), ValueError, "contiguous"),
    (dict(cache=cache(nkv=1)), ValueError, "KV heads"),
    (dict(cache=cache(rows=1)), ValueError, "batch"),
    (dict(start=n64(0)), ValueError, "start"),
    (dict(lengths=torch.zeros(2, dtype=torch.bool)), TypeError, "lengths"),
])
def test_quantize_refuses(kw, error, match):
    a = dict(k=torch.zeros(2, 2, 5, 64, dtype=BF), v=torch.zeros(2, 2, 5, 64, dtype=BF), cache=cache())
    a.update(kw)
    with pytest.raises(error, match=match):
        quantize_kv(**a)


def test_dequantize_refuses():
    with pytest.raises(RuntimeError, match="CUDA"):
        dequantize_kv(cache())
    with pytest.raises(TypeError, match="QuantKV"):
        dequantize_kv(plain())
    for n in (17, -1):
        with pytest.raises(ValueError, match="positions"):
            dequantize_kv(cache(), n)


def attn_call(behind=False, **kw):
    a = dict(q=torch.zeros(2, 4, 1, 64, dtype=BF), cache=cache(), seqlen=n64(0, 1), scale=1.0)
    if behind:
        a["prefix"] = SharedPrefix(cache(3, n=9), n64(1, 2, 3), n64(0, -1))
    a.update(kw)
    return (prefix_gqa_attn if "prefix" in a else quant_gqa_attn)(**a)


@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("kw,error,match", [
    (dict(), RuntimeError, "CUDA"),
    (dict(q=torch.zeros(2, 4, 1, 64)), ValueError, "bf16"),
    (dict(q=torch.zeros(2, 4, 2, 64, dtype=BF)), ValueError, "bf16"),
    (dict(q=torch.zeros(2, 4, 1, 128, dtype=BF)), ValueError, "heads of"),
    (dict(q=torch.zeros(2, 3, 1, 64, dtype=BF)), ValueError, "divisible"),
    (dict(q=torch.zeros(3, 4, 1, 64, dtype=BF), seqlen=n64(0, 1, 2)), ValueError, "batch"),
    (dict(window=0), ValueError, "window"),
    (dict(window=-3), ValueError, "window"),
    (dict(seqlen=n64(1)), ValueError, "seqlen"),
    (dict(row_map=n64(1)), ValueError, "row_map"),
    (dict(cache=(1, 2)), TypeError, "QuantKV"),
])
def test_attention_refuses(prefix, kw, error, match):
    with pytest.raises(error, match=match):
        attn_call(prefix, **kw)


@pytest.mark.parametrize("prefix,error,match", [
    (SharedPrefix(plain(3), n64(1, 2, 3), n64(0, 1)), TypeError, "behind"),
    (SharedPrefix(cache(3, nkv=1), n64(1, 2, 3), n64(0, 1)), ValueError, "prefixes"),
    (SharedPrefix(cache(3, d=128), n64(1, 2, 3), n64(0, 1)), ValueError, "prefixes"),
    (SharedPrefix(cache(3), n64(1, 2), n64(0, 1)), ValueError, "length"),
    (SharedPrefix(cache(3), n64(1, 2, 3), n64(0)), ValueError, "of"),
    (SharedPrefix(cache(3), n64(1, 2, 3), torch.zeros(2)), TypeError, "of"),
])
def test_prefixes_refused(prefix, error, match):
    with pytest.raises(error, match=match):
        attn_call(prefix=prefix)


def c_attn(**kw):
    a = dict(q=FAKE, batch=2, nq=4, nkv=2, d=64, k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, rows=2, n=128, seqlen=FAKE, rm=None,
             pk=None, pv=None, pks=None, pvs=None, p=0, pn=0, plen=None, of=None, once=-1, window=0, scale=1.0, out=FAKE,
             ws=FAKE, nbytes=1 << 40, stream=None)
    a.update(kw)
    return _lib.call("ma_cache_attn", *a.values())


PRE = dict(pk=FAKE, pv=FAKE, pks=FAKE, pvs=FAKE, p=3, pn=100, plen=FAKE, of=FAKE)


@pytest.mark.parametrize("kw,match", [
    (dict(d=96), "head_dim"), (dict(nq=5), "query heads"), (dict(nq=34), "query heads"), (dict(nkv=0), "query heads"),
    (dict(batch=-1), "batch"), (dict(batch=40000), "batch"), (dict(rows=1), "cache sizes"), (dict(n=0), "cache sizes"),
    (dict(window=-1), "window"), (dict(scale=float("nan")), "scale"), (dict(scale=3e38), "scale"),
    (dict(q=None), "null"), (dict(vs=None), "null"), (dict(ks=None), "null"), (dict(out=None), "null"),
    (dict(k=FAKE + 8), "aligned"), (dict(ws=FAKE + 4), "aligned"), (dict(n=4096, ws=None), "workspace"),
    (dict(n=4096, nbytes=100), "workspace"),
    (dict(PRE, of=None), "null"), (dict(PRE, pks=None), "kind"), (dict(PRE, ks=None, vs=None), "kind"),
    (dict(PRE, pn=0), "prefixes"), (dict(PRE, p=-1), "prefixes"), (dict(PRE, p=70000), "prefixes"),
    (dict(PRE, pk=FAKE + 8), "aligned"),
    (dict(PRE, once=1, window=5), "each row"), (dict(PRE, once=1, p=65), "each row"),
])
def test_c_attention_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        c_attn(**kw)


def test_c_attention_workspace():
    lib = _lib.load()
    need = lambda *a: int(lib.ma_cache_attn_workspace_bytes(*a, *(() if len(a) == 10 else (1, -1))))  # noqa: E731
    assert need(1, 32, 4, 64, 4096, 0, 0, 0) > 0
    assert need(1, 32, 4, 64, 128, 0, 0, 0) == 0  # one split: nothing to join
    assert need(0, 32, 4, 64, 4096, 0, 0, 0) == 0
    assert need(1, 32, 4, 96, 4096, 0, 0, 0) == 0
    # a window past every distance is none
    assert need(4, 32, 4, 64, 4096, 2, 1000, 2 ** 62) == need(4, 32, 4, 64, 4096, 2, 1000, 0) > 0
    # a prefix that is read once is a part of its own
    once = lambda kind, form, b=64, n=2000, p=2: need(b, 32, 4, 64, 128, p, n, 0, kind, form)  # noqa: E731
    assert once(1, -1) == once(1, 1) != once(1, 0)
    assert once(0, -1, n=1000) == once(0, 1, n=1000) and once(1, -1, n=1000) == once(1, 0, n=1000)  # (by its bytes)
    assert once(1, -1, b=4) == once(1, 0, b=4) and once(1, -1, p=64) == once(1, 0, p=64)  # (by the rows behind it)
    assert once(1, 1, p=65) == 0  # (refused)


@pytest.mark.parametrize("entry,args,match", [
    ("ma_quant_kv", dict(d=80), "head_dim"), ("ma_quant_kv", dict(t=-1), "bad sizes"),
    ("ma_quant_kv", dict(k=None), "null"), ("ma_quant_kv", dict(kc=None), "null"),
    ("ma_quant_kv", dict(kc=FAKE + 8), "aligned"), ("ma_quant_kv", dict(batch=3), "cache sizes"),
    ("ma_quant_kv", dict(t=1 << 40), "too large"),
    ("ma_dequant_kv", dict(t=17), "positions"), ("ma_dequant_kv", dict(out=None), "outputs"),
    ("ma_dequant_kv", dict(out=FAKE + 2), "outputs"), ("ma_dequant_kv", dict(ks=None), "null"),
])
def test_c_copies_refuse(entry, args, match):
    a = dict(k=FAKE, kc=FAKE, ks=FAKE, batch=2, t=5, nkv=2, d=64, rows=2, n=16, out=FAKE)
    a.update(args)
    with pytest.raises(ValueError, match=match):
        if entry == "ma_quant_kv":
            _lib.call(entry, a["k"], 640, 320, 64, FAKE, 640, 320, 64, a["batch"], a["t"], a["nkv"], a["d"], None, None,
                      None, a["kc"], FAKE, a["ks"], FAKE, a["rows"], a["n"], None)
        else:
            _lib.call(entry, a["kc"], FAKE, a["ks"], FAKE, a["rows"], a["n"], a["batch"], a["t"], a["nkv"], a["d"], None,
                      a["out"], FAKE, None)


C_QKV_REFUSED = [
    (dict(d=32), ValueError, "head_dim"), (dict(nq=3), ValueError, "query heads"), (dict(ld=100), ValueError, "stride"),
    (dict(rot=66), ValueError, "rotary_dim"), (dict(rot=7), ValueError, "rotary_dim"), (dict(cos=None), ValueError, "tables"),
    (dict(n_pos=0), ValueError, "tables"), (dict(ld_cs=30), ValueError, "tables"), (dict(w_dt=9), TypeError, "dtype"),
    (dict(qw=None), ValueError, "norm weight"), (dict(qkv=None), ValueError, "null"), (dict(out=FAKE + 8), ValueError, "aligned"),
    (dict(batch=3), ValueError, "cache sizes"), (dict(batch=1 << 30, rm=FAKE), ValueError, "too large"),
]


def c_qkv(**kw):
    a = dict(qkv=FAKE, ld=512, batch=2, nq=4, nkv=2, d=64, qw=FAKE, kw=FAKE, w_dt=0, cos=FAKE, sin=FAKE, dt=0, ld_cs=32,
             n_pos=16, rot=32, eps=1e-6, seqlen=FAKE, at=None, rm=None, kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, rows=2, n=16,
             out=FAKE, stream=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error,match", C_QKV_REFUSED)
def test_c_qkv_refuses(kw, error, match):
    with pytest.raises(error, match=match):
        _lib.call("ma_quant_qkv", *c_qkv(**kw).values())


@pytest.mark.parametrize("kw,error,match", C_QKV_REFUSED + [
    (dict(window=-1), ValueError, "window"), (dict(scale=float("inf")), ValueError, "scale"),
    (dict(nq=34), ValueError, "query heads"), (dict(n=4096, ws=None), ValueError, "workspace"),
    (dict(n=4096, nbytes=99), ValueError, "workspace"), (dict(ws=FAKE + 4), ValueError, "aligned"),
    (dict(ks=None), ValueError, "null"), (dict(kc=FAKE + 8), ValueError, "aligned"), (dict(seqlen=None), ValueError, "null"),
])
def test_c_fused_attention_refuses(kw, error, match):
    a = c_qkv()
    out, stream = a.pop("out"), a.pop("stream")
    a.update(window=0, scale=1.0, out=out, ws=FAKE, nbytes=1 << 40, stream=stream)
    a.update(kw)
    with pytest.raises(error, match=match):
        _lib.call("ma_quant_attn", *a.values())
