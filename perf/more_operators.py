"""Timing cases of decoding over a quantised cache and over shared prefixes.

A quantised cache holds, per (row, KV head, position) and for K and V each,
``head_dim`` e4m3 codes and one power of two (e8m0): the least ``2^e`` with which
the largest value is at most 448.  Five operators write and read it:

* ``qkv``: ``apply_qkv_quant``, QK RMSNorm and rotary positions of one token a row
  and the quantising store of its K and V;
* ``quant``: ``quantize_kv``, the K and V of whole prompts into the cache;
* ``dequant``: ``dequantize_kv``, cached positions back as bf16;
* ``attn``: ``quant_gqa_attn``, one query token a row over the quantised cache;
* ``prefix``: ``prefix_gqa_attn``, the same for rows whose sequences begin with one
  of a few long prefixes (a system prompt, a document), each held once and read once
  for all of its rows, in bf16 or quantised.

``run`` makes these calls where ``own`` is true and computes the same values in
elementary torch operations where it is false.  Codes and scales are returned as
the float8 tensors that they are kept in.
"""

import functools
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
THETA = 10000.0
# (query heads, KV heads, head_dim): the attention of the benchmark's two decoders
HEADS = {"64": (32, 4, 64), "128": (16, 4, 128)}


def listed():
    return [
        # one stream's new token behind a 4096-token context: latency of the smallest call
        dict(name="qkv_b1", kind="qkv", batch=1, length=4096, heads="64", rot=32),
        # the widest serving step, the whole head rotated
        dict(name="qkv_b256_128", kind="qkv", batch=256, length=512, heads="128", rot=128),
        # a few tokens of one prompt
        dict(name="quant_b1_t7", kind="quant", batch=1, length=7, heads="64"),
        # the prompts of a whole batch, of different lengths
        dict(name="quant_b32_t4096", kind="quant", batch=32, length=4096, heads="64"),
        # one sequence of an odd length read back
        dict(name="dequant_b1_l1001_128", kind="dequant", batch=1, length=1001, heads="128"),
        # a whole batch read back
        dict(name="dequant_b32_l4096", kind="dequant", batch=32, length=4096, heads="64"),
        # one stream at the benchmark's context
        dict(name="attn_b1_l4096", kind="attn", batch=1, length=4096, heads="64", window=0),
        # a serving batch at the benchmark's context, rows of different lengths
        dict(name="attn_b32_l4096", kind="attn", batch=32, length=4096, heads="64", window=0),
        # a few long contexts
        dict(name="attn_b8_l32768_128", kind="attn", batch=8, length=32768, heads="128", window=0),
        # odd sizes: five rows, two prefixes, a bf16 cache
        dict(name="prefix_b5_p1001_128", kind="prefix", batch=5, groups=2, prefix=1001, length=37, heads="128",
             quant=False, window=0),
        # a serving batch behind one document, a bf16 cache
        dict(name="prefix_b32_p8192", kind="prefix", batch=32, groups=1, prefix=8192, length=512, heads="64",
             quant=False, window=0),
        # a wide batch behind four documents, a quantised cache
        dict(name="prefix_b64_p16384_e4m3", kind="prefix", batch=64, groups=4, prefix=16384, length=1024, heads="64",
             quant=True, window=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["qkv", "quant", "dequant", "attn", "attn", "prefix", "prefix"])
    heads = rng.choice(["64", "128"])
    d = HEADS[heads][2]
    batch = _log_int(rng, 1, 64)
    if kind == "qkv":
        batch = _log_int(rng, 1, 256)
        return dict(kind=kind, batch=batch, length=min(_log_int(rng, 16, 4096), 131072 // batch), heads=heads,
                    rot=rng.choice([d, d // 2, d // 2 - 12, d // 4]))
    if kind in ("quant", "dequant"):
        return dict(kind=kind, batch=batch, length=_log_int(rng, 1, 4096 * 2048 // (batch * d)), heads=heads)
    if kind == "attn":
        return dict(kind=kind, batch=batch, length=_log_int(rng, 1, min(32768, 2 ** 25 // (batch * d))), heads=heads,
                    window=rng.choice([0, 0, 512]))
    prefix = _log_int(rng, 64, 16384)
    batch = max(1, min(batch, 2 ** 25 // (d * prefix)))
    return dict(kind=kind, batch=batch, groups=rng.choice([1, 1, 2, 3]), prefix=prefix, length=_log_int(rng, 1, 1024),
                heads=heads, quant=rng.random() < 0.5, window=rng.choice([0, 0, 0, 512]))


# ---------------------------------------------------------------------------
# Inputs, from the seed alone.
# ---------------------------------------------------------------------------
class _Make:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(1_000_003 * int(seed) + 41)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=torch.bfloat16)

    def rand(self, *shape):
        return torch.rand(shape, generator=self.g, device=DEV)

    def lengths(self, n, length):
        """Half of ``length`` to ``length`` each, the first the longest."""
        x = torch.randint((length + 1) // 2, length + 1, (n,), generator=self.g, device=DEV)
        x[0] = length
        return x

    def kv(self, rows, nkv, n, d):
        """K and V as attention meets them: some of K's channels larger than others, V's size differing by token."""
        k = self.normal(rows, nkv, n, d) * (self.rand(nkv, 1, d) * 2 + 0.25).bfloat16()
        v = self.normal(rows, nkv, n, d) * torch.exp2(4 * self.rand(rows, nkv, n, 1) - 3).bfloat16()
        return k, v


def _tables(n_pos, rot):
    """cos / sin ``[n_pos, rot]`` in bf16, angles in 64 bits, the frequencies in both halves of a row."""
    inv = THETA ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    a = torch.arange(n_pos, device=DEV, dtype=torch.float64).unsqueeze(1) * inv
    a = torch.cat([a, a], -1)
    return a.cos().bfloat16(), a.sin().bfloat16()


def _max_len(case):
    return case["length"] + 128


def prepare(case, seed):
    c, m = case, _Make(seed)
    b = c["batch"]
    nq, nkv, d = HEADS[c["heads"]]
    s = dict(case=case)
    if c["kind"] == "quant":
        # as a prompt's projection leaves them: positions before heads
        k, v = m.kv(b, nkv, c["length"], d)
        s["k"], s["v"] = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
        s["lengths"] = m.lengths(b, c["length"])
        s["cache"] = _encode(*m.kv(b, nkv, _max_len(c), d))
        return s
    if c["kind"] == "dequant":
        s["cache"] = _encode(*m.kv(b, nkv, _max_len(c), d))
        return s
    s["seqlen"] = m.lengths(b, c["length"]) - 1  # the last position that holds a token
    cache = m.kv(b, nkv, _max_len(c), d)
    s["cache"] = _encode(*cache) if c["kind"] != "prefix" or c["quant"] else cache
    if c["kind"] == "qkv":
        s["qkv"] = m.normal(b, (nq + 2 * nkv) * d)
        s["qw"], s["kw"] = m.rand(d) + 0.5, m.rand(d) + 0.5
        s["cos"], s["sin"] = _tables(_max_len(c), c["rot"])
        return s
    s["q"] = m.normal(b, nq, 1, d)
    if c["kind"] == "prefix":
        shared = m.kv(c["groups"], nkv, c["prefix"], d)
        s["shared"] = _encode(*shared) if c["quant"] else shared
        s["shared_len"] = m.lengths(c["groups"], c["prefix"])
        # most rows have a prefix; the first row has the first
        s["of"] = torch.randint(0, c["groups"], (b,), generator=m.g, device=DEV)
        s["of"] = torch.where(m.rand(b) < 0.05, -1, s["of"])
        s["of"][0] = 0
    return s


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)[state["case"]["kind"]](state)


@functools.lru_cache(maxsize=None)
def _kernels():
    import __graft_entry__

    __graft_entry__.load_package()
    from maple_amd import kernels

    return kernels


def _own_qkv(s):
    c = s["case"]
    nq, nkv, d = HEADS[c["heads"]]
    q = _kernels().apply_qkv_quant(s["qkv"], s["qw"], s["kw"], s["cos"], s["sin"], _kernels().QuantKV(*s["cache"]),
                                   s["seqlen"], num_heads=nq, num_kv_heads=nkv, head_dim=d, rotary_dim=c["rot"],
                                   eps=EPS)
    return q, s["cache"]


def _own_quant(s):
    _kernels().quantize_kv(s["k"], s["v"], _kernels().QuantKV(*s["cache"]), lengths=s["lengths"])
    return s["cache"]


def _own_dequant(s):
    return _kernels().dequantize_kv(_kernels().QuantKV(*s["cache"]), s["case"]["length"])


def _own_attn(s):
    c = s["case"]
    return _kernels().quant_gqa_attn(s["q"], _kernels().QuantKV(*s["cache"]), s["seqlen"],
                                     scale=HEADS[c["heads"]][2] ** -0.5, window=c["window"] or None)


def _own_prefix(s):
    c, k = s["case"], _kernels()
    kv = k.QuantKV if c["quant"] else k.KV
    return k.prefix_gqa_attn(s["q"], kv(*s["cache"]), s["seqlen"],
                             k.SharedPrefix(kv(*s["shared"]), s["shared_len"], s["of"]),
                             scale=HEADS[c["heads"]][2] ** -0.5, window=c["window"] or None)


_own = {"qkv": _own_qkv, "quant": _own_quant, "dequant": _own_dequant, "attn": _own_attn, "prefix": _own_prefix}


def _encode_one(x):
    """Codes and scales of bf16 rows ``[..., D]``."""
    top = x.abs().amax(-1).view(torch.int16).int()
    # 448 is 1.75 2^8: a largest value of mantissa past 1.75 needs one power of two more
    e = (((top + 31) >> 7) - 8).clamp(1, 246)
    y = x.float() * ((254 - e) << 23).view(torch.float32).unsqueeze(-1)
    return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), e.to(torch.uint8).view(torch.float8_e8m0fnu)


def _encode(k, v):
    """A quantised cache ``(k, v, k_scale, v_scale)`` of bf16 K and V."""
    (kc, ks), (vc, vs) = _encode_one(k), _encode_one(v)
    return kc, vc, ks, vs


def _decode(codes, scale):
    """The values in 32 bits."""
    return codes.float() * (scale.view(torch.uint8).int() << 23).view(torch.float32).unsqueeze(-1)


def _plain_qkv(s):
    c = s["case"]
    nq, nkv, d = HEADS[c["heads"]]
    b, rot = c["batch"], c["rot"]
    x = s["qkv"].float().view(b, nq + 2 * nkv, d)
    cos, sin = (s[n].float()[s["seqlen"]].unsqueeze(1) for n in ("cos", "sin"))
    h = rot // 2

    def norm_rotate(y, w):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
        lo, hi = y[..., :h], y[..., h:rot]
        return torch.cat([lo * cos[..., :h] - hi * sin[..., :h], hi * cos[..., h:] + lo * sin[..., h:], y[..., rot:]],
                         -1).bfloat16()

    q = norm_rotate(x[:, :nq], s["qw"])
    k = norm_rotate(x[:, nq:nq + nkv], s["kw"])
    v = s["qkv"].view(b, nq + 2 * nkv, d)[:, nq + nkv:]
    rows = torch.arange(b, device=DEV)
    for to, new in zip(s["cache"], _encode(k, v)):
        to.view(torch.uint8)[rows, :, s["seqlen"]] = new.view(torch.uint8)
    return q.unsqueeze(2), s["cache"]


def _plain_quant(s):
    t = s["case"]["length"]
    there = torch.arange(t, device=DEV) < s["lengths"].unsqueeze(1)
    for to, new in zip(s["cache"], _encode(s["k"], s["v"])):
        old = to.view(torch.uint8)[:, :, :t]
        keep = there.view(there.shape[0], 1, t, *[1] * (old.ndim - 3))
        old.copy_(torch.where(keep, new.view(torch.uint8), old))
    return s["cache"]


def _plain_dequant(s):
    n = s["case"]["length"]
    k, v, ks, vs = (t[:, :, :n] for t in s["cache"])
    return _decode(k, ks).bfloat16(), _decode(v, vs).bfloat16()


def _softmax_v(q, k, v, seen):
    """``q [B, nkv, g, D]``, ``k`` / ``v [B, nkv, n, D]``, ``seen [B, n]``, all in 32 bits."""
    x = (q @ k.transpose(-1, -2)).mul_(q.shape[-1] ** -0.5)
    x.masked_fill_(~seen.view(seen.shape[0], 1, 1, -1), -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    return (x @ v) / x.sum(-1, keepdim=True)


def _values(cache):
    return (_decode(cache[0], cache[2]), _decode(cache[1], cache[3])) if len(cache) == 4 else (
        cache[0].float(), cache[1].float())


def _plain_attn(s):
    c = s["case"]
    nq, nkv, d = HEADS[c["heads"]]
    b = c["batch"]
    k, v = _values(s["cache"])
    j = torch.arange(k.shape[2], device=DEV)
    n = s["seqlen"].unsqueeze(1)
    seen = j <= n
    if c["window"]:
        seen = seen & (j > n - c["window"])
    return _softmax_v(s["q"].float().view(b, nkv, nq // nkv, d), k, v, seen).reshape(b, nq, 1, d).bfloat16()


def _plain_prefix(s):
    """The prefix laid before each row's own positions."""
    c = s["case"]
    nq, nkv, d = HEADS[c["heads"]]
    b = c["batch"]
    of = s["of"].clamp(min=0)
    size = torch.where(s["of"] >= 0, s["shared_len"][of], 0).unsqueeze(1)
    k, v = (torch.cat([p[of], x], 2) for p, x in zip(_values(s["shared"]), _values(s["cache"])))
    j = torch.arange(k.shape[2], device=DEV).unsqueeze(0)
    behind = j - c["prefix"]  # an own position
    at = torch.where(behind < 0, j, behind + size)  # where it stands in the sequence
    last = size + s["seqlen"].unsqueeze(1)
    seen = ((behind >= 0) | (j < size)) & (at <= last)
    if c["window"]:
        seen = seen & (at > last - c["window"])
    return _softmax_v(s["q"].float().view(b, nkv, nq // nkv, d), k, v, seen).reshape(b, nq, 1, d).bfloat16()


_plain = {"qkv": _plain_qkv, "quant": _plain_quant, "dequant": _plain_dequant, "attn": _plain_attn,
          "prefix": _plain_prefix}


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------
def work(case):
    c = case
    nq, nkv, d = HEADS[c["heads"]]
    b = c["batch"]
    mean = lambda n, rows: n if rows == 1 else (n + 0.75 * n * (rows - 1)) / rows  # noqa: E731  (half of n to n)
    if c["kind"] == "qkv":
        return {"bytes": b * ((nq + 2 * nkv) * d * 2 + nq * d * 2 + 2 * nkv * (d + 1) + c["rot"] * 4),
                "flops": b * (nq + nkv) * d * 10}
    if c["kind"] == "quant":
        return {"bytes": b * mean(c["length"], b) * 2 * nkv * (2 * d + d + 1), "flops": 0}
    if c["kind"] == "dequant":
        return {"bytes": b * c["length"] * 2 * nkv * (2 * d + d + 1), "flops": 0}
    length = mean(c["length"], b)
    ends = 2 * b * nq * d * 2  # q and the output
    if c["kind"] == "attn":
        span = min(length, c["window"]) if c["window"] else length
        return {"bytes": b * span * 2 * nkv * (d + 1) + ends, "flops": 4 * b * nq * d * span}
    prefix = mean(c["prefix"], c["groups"])
    if c["window"]:
        length = min(length, c["window"])
        prefix = min(prefix, c["window"] - length)
    groups = min(c["groups"], b)
    return {"bytes": (groups * prefix + b * length) * 2 * nkv * (d + 1 if c["quant"] else 2 * d) + ends,
            "flops": 4 * b * nq * d * (prefix + length)}


# ---------------------------------------------------------------------------
# The same values in 64 bits, row by row.
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["batch"] * (case["length"] + case.get("prefix", 0)) > 2 ** 21:
        return None
    return {"qkv": _exact_qkv, "quant": _exact_quant, "dequant": _exact_dequant, "attn": _exact_attn,
            "prefix": _exact_attn}[case["kind"]](prepare(case, seed), case)


def _power(x):
    """The scale's exponent of rows in 64 bits: the least with which the largest value is at most 448."""
    top = x.abs().amax(-1)
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -117) / 448.0))
    e = torch.where(torch.exp2(e - 1) * 448.0 >= top, e - 1, e)
    return torch.where(torch.exp2(e) * 448.0 < top, e + 1, e).clamp(-126, 119)


def _wide(codes, scale):
    """Cached values in 64 bits."""
    p = scale.view(torch.uint8).double() - 127.0
    return codes.double() * torch.exp2(p).unsqueeze(-1)


def _exact_qkv(s, c):
    nq, nkv, d = HEADS[c["heads"]]
    rot, half = c["rot"], c["rot"] // 2
    x = s["qkv"].double().view(c["batch"], nq + 2 * nkv, d)
    out = [s["cache"][i].double() for i in range(4)]
    q = torch.empty(c["batch"], nq, 1, d, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["seqlen"].tolist()):
        cos, sin = s["cos"][n].double(), s["sin"][n].double()
        turned = []
        for rows, w in ((x[b, :nq], s["qw"]), (x[b, nq:nq + nkv], s["kw"])):
            y = rows / torch.sqrt((rows * rows).sum(-1, keepdim=True) / d + EPS) * w.double()
            z = y.clone()
            z[:, :half] = y[:, :half] * cos[:half] - y[:, half:rot] * sin[:half]
            z[:, half:rot] = y[:, half:rot] * cos[half:] + y[:, :half] * sin[half:]
            turned.append(z)
        q[b, :, 0] = turned[0]
        for i, new in enumerate((turned[1], x[b, nq + nkv:])):
            p = _power(new)
            out[i][b, :, n] = new / torch.exp2(p).unsqueeze(-1)
            out[2 + i][b, :, n] = torch.exp2(p)
    return q, tuple(out)


def _exact_quant(s, c):
    out = [t.double() for t in s["cache"]]
    for b, n in enumerate(s["lengths"].tolist()):
        for i, new in enumerate((s["k"], s["v"])):
            x = new[b, :, :n].double()
            p = _power(x)
            out[i][b, :, :n] = x / torch.exp2(p).unsqueeze(-1)
            out[2 + i][b, :, :n] = torch.exp2(p)
    return tuple(out)


def _exact_dequant(s, c):
    k, v, ks, vs = (t[:, :, :c["length"]] for t in s["cache"])
    return _wide(k, ks), _wide(v, vs)


def _rows_wide(cache, row, lo, hi):
    if len(cache) == 2:
        return cache[0][row, :, lo:hi].double(), cache[1][row, :, lo:hi].double()
    return _wide(cache[0][row, :, lo:hi], cache[2][row, :, lo:hi]), _wide(cache[1][row, :, lo:hi],
                                                                          cache[3][row, :, lo:hi])


def _exact_attn(s, c):
    nq, nkv, d = HEADS[c["heads"]]
    out = torch.empty(c["batch"], nq, 1, d, dtype=torch.float64, device=DEV)
    of = s["of"].tolist() if "of" in s else [-1] * c["batch"]
    sizes = s["shared_len"].tolist() if "of" in s else []
    for b, n in enumerate(s["seqlen"].tolist()):
        k, v = _rows_wide(s["cache"], b, 0, n + 1)
        if of[b] >= 0:
            pk, pv = _rows_wide(s["shared"], of[b], 0, sizes[of[b]])
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        if c["window"]:
            k, v = k[:, -c["window"]:], v[:, -c["window"]:]
        q = s["q"][b, :, 0].double().view(nkv, nq // nkv, d)
        p = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(d), -1)
        out[b, :, 0] = torch.matmul(p, v).view(nq, d)
    return out
