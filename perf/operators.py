"""Timing cases of decoding with drafted token trees.

A draft (a small model, extra heads, a table of n-grams) proposes a tree of
tokens per sequence; one pass of the model scores all of them and the branch
that the model's own law accepts is kept.  Four operators carry that step:

* ``qkv``: ``apply_qkv_tree``, QK RMSNorm, rotary positions by depth in the
  tree (half or interleaved layout, all or part of the head, any table) and the
  store of the nodes' K and V behind the sequence;
* ``attn``: ``tree_attention``, every node over its sequence and its own
  ancestors;
* ``verify``: ``verify_tree``, the walk down the tree that accepts drafted
  tokens against the target's law with given uniforms, and the last draw;
* ``commit``: ``commit_tree``, the accepted nodes' K and V moved together.

``run`` makes these calls where ``own`` is true and computes the same values in
elementary torch operations where it is false.

A tree is ``parents [batch, nodes]`` (int32): node 0 is the last token of the
sequence (parent -1), every other node's parent comes before it, and -1 marks
padding (rows have different numbers of nodes).
"""

import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6
THETA = 10000.0
VOCAB = 151936
# (query heads, KV heads, head_dim): the attention of the benchmark's two decoders
HEADS = {"64": (32, 4, 64), "128": (16, 4, 128)}


def listed():
    return [
        # one stream with a short draft: latency of the smallest call
        dict(name="qkv_b1_t8", kind="qkv", batch=1, nodes=8, length=1024, heads="64", rot=32, interleaved=False),
        # a serving batch with trees of 32 nodes, half of the head rotated
        dict(name="qkv_b32_t32", kind="qkv", batch=32, nodes=32, length=2048, heads="64", rot=32, interleaved=False),
        # large ragged trees far into a long context, the whole head rotated in pairs
        dict(name="qkv_b8_t61_far", kind="qkv", batch=8, nodes=61, length=32768, heads="128", rot=128, interleaved=True),
        # one stream with a short draft behind a 4096-token context
        dict(name="attn_b1_t8_l4096", kind="attn", batch=1, nodes=8, length=4096, heads="64", window=0),
        # a serving batch, rows of different lengths, trees of 32 nodes
        dict(name="attn_b32_t32_l4096", kind="attn", batch=32, nodes=32, length=4096, heads="64", window=0),
        # a few long contexts with the largest trees
        dict(name="attn_b2_t64_l32768", kind="attn", batch=2, nodes=64, length=32768, heads="128", window=0),
        # odd sizes on a sliding-window layer
        dict(name="attn_b7_t23_w512", kind="attn", batch=7, nodes=23, length=3001, heads="128", window=512),
        # one stream, greedy: a drafted token is kept where it is the argmax
        dict(name="verify_b1_t8_greedy", kind="verify", batch=1, nodes=8, vocab=VOCAB, top_k=1, top_p=1.0, temp=1.0,
             probs=False),
        # a mid-sized batch against the draft model's probabilities
        dict(name="verify_b8_t13_probs", kind="verify", batch=8, nodes=13, vocab=VOCAB, top_k=50, top_p=0.95, temp=0.8,
             probs=True),
        # the widest: a serving batch with trees picked without probabilities
        dict(name="verify_b32_t32", kind="verify", batch=32, nodes=32, vocab=VOCAB, top_k=64, top_p=0.9, temp=0.7,
             probs=False),
        # one stream's accepted branch in all layers of the benchmark's decoder
        dict(name="commit_b1_t8", kind="commit", batch=1, nodes=8, length=1024, heads="64", layers=24),
        # the same of a batch with larger trees
        dict(name="commit_b32_t32", kind="commit", batch=32, nodes=32, length=64, heads="64", layers=24),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["qkv", "attn", "attn", "verify", "verify", "commit"])
    nodes = _log_int(rng, 1, 64)
    heads = rng.choice(["64", "128"])
    batch = _log_int(rng, 1, 32)
    if kind == "qkv":
        d = HEADS[heads][2]
        batch = min(batch, max(1, 1024 // nodes))
        length = min(_log_int(rng, 64, 32768), 262144 // batch)
        return dict(kind=kind, batch=batch, nodes=nodes, length=length, heads=heads,
                    rot=rng.choice([d, d // 2, d // 2 - 12, d // 4]), interleaved=rng.random() < 0.5)
    if kind == "attn":
        length = _log_int(rng, 1, 32768)
        batch = min(batch, max(1, 4194304 // (nodes * length)), max(1, 131072 // length))
        return dict(kind=kind, batch=batch, nodes=nodes, length=length, heads=heads, window=rng.choice([0, 0, 512]))
    if kind == "verify":
        probs = rng.random() < 0.5
        batch = min(batch, max(1, (256 if probs else 1024) // nodes))
        return dict(kind=kind, batch=batch, nodes=nodes, vocab=rng.choice([VOCAB, VOCAB, 100003, 32000]),
                    top_k=rng.choice([1, 7, 20, 50, 64]), top_p=rng.choice([1.0, 0.95, 0.8]),
                    temp=rng.choice([1.0, 0.7, 1.3]), probs=probs)
    return dict(kind=kind, batch=batch, nodes=max(2, nodes), length=_log_int(rng, 1, 2048 // batch), heads=heads,
                layers=rng.choice([4, 12, 24]))


# ---------------------------------------------------------------------------
# Inputs, from the seed alone.
# ---------------------------------------------------------------------------
class _Make:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(1_000_003 * int(seed) + 29)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=torch.bfloat16)

    def rand(self, *shape):
        return torch.rand(shape, generator=self.g, device=DEV)

    def lengths(self, batch, length):
        """Positions in the cache per row: half of ``length`` to ``length``, the first row the longest."""
        n = torch.randint((length + 1) // 2, length + 1, (batch,), generator=self.g, device=DEV)
        n[0] = length
        return n

    def parents(self, batch, nodes):
        """Trees that grow like drafted ones: a node hangs on the one before it or on a random earlier one; past the
        first row, a row keeps half to all of its nodes."""
        i = torch.arange(nodes, device=DEV)
        p = torch.where(self.rand(batch, nodes) < 0.5, i - 1, (self.rand(batch, nodes) * i).long())
        n = torch.randint((nodes + 1) // 2, nodes + 1, (batch, 1), generator=self.g, device=DEV)
        n[0] = nodes
        p = torch.where(i < n, p, -1)
        p[:, 0] = -1
        return p.int()


def _tables(n_pos, rot):
    """cos / sin ``[n_pos, rot]`` in bf16, angles in 64 bits, the frequencies in both halves of a row."""
    inv = THETA ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    a = torch.arange(n_pos, device=DEV, dtype=torch.float64).unsqueeze(1) * inv
    a = torch.cat([a, a], -1)
    return a.cos().bfloat16(), a.sin().bfloat16()


def _max_len(case):
    return case["length"] + (64 if case["kind"] == "commit" else 128)


def prepare(case, seed):
    c, m = case, _Make(seed)
    b, t = c["batch"], c["nodes"]
    s = dict(case=case, parents=m.parents(b, t))
    if c["kind"] == "verify":
        return _prepare_verify(s, m)
    nq, nkv, d = HEADS[c["heads"]]
    s["seqlen"] = m.lengths(b, c["length"])
    cache = lambda: m.normal(b, nkv, _max_len(c), d)  # noqa: E731
    if c["kind"] == "commit":
        reach, _, _ = _tree(s["parents"])
        i = torch.arange(t, device=DEV)
        last = torch.minimum((m.rand(b) * t).long(), (s["parents"] >= 0).sum(1))
        on = reach[torch.arange(b, device=DEV), last] > 0  # the nodes on the way to the last accepted one
        path = torch.where(on, i, t).sort(1).values
        s["path"] = torch.where(path < t, path, -1).int()
        s["accepted"] = (on.sum(1) - 1).int()
        s["k"] = [cache() for _ in range(c["layers"])]
        s["v"] = [cache() for _ in range(c["layers"])]
        return s
    s["k"], s["v"] = cache(), cache()
    if c["kind"] == "attn":
        s["q"] = m.normal(b, t, nq, d)
        return s
    s["qkv"] = m.normal(b, t, (nq + 2 * nkv) * d)
    s["qw"], s["kw"] = m.rand(d) + 0.5, m.rand(d) + 0.5
    s["cos"], s["sin"] = _tables(_max_len(c), c["rot"])
    return s


def _prepare_verify(s, m):
    """Logits with a few likely tokens a row; a drafted token is one of its parent's likely ones, or drawn from the
    draft's probabilities, which are the parent's with noise."""
    c = s["case"]
    b, t, v = c["batch"], c["nodes"], c["vocab"]
    x = torch.randn(b, t, v, generator=m.g, device=DEV)
    x.mul_(2.0)
    likely = torch.randint(0, v, (b, t, 6), generator=m.g, device=DEV)
    x.scatter_(2, likely, 9.0 + 4.0 * m.rand(b, t, 6))
    s["logits"] = x.bfloat16()
    up = s["parents"].long().clamp(min=0)
    mine = torch.gather(likely, 1, up.unsqueeze(-1).expand(b, t, 6))
    rank = (m.rand(b, t, 1) * 6).long()
    s["tokens"] = torch.gather(mine, 2, rank).squeeze(-1)
    s["probs"] = None
    if c["probs"]:
        x = torch.gather(x, 1, up.unsqueeze(-1).expand(b, t, v))
        x.add_(torch.randn(b, t, v, generator=m.g, device=DEV), alpha=0.5)
        s["probs"] = torch.softmax(x / c["temp"], -1)
        s["tokens"] = torch.multinomial(s["probs"].view(b * t, v), 1, generator=m.g).view(b, t)
    s["uniform"] = m.rand(b, t)
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
    q = _kernels().apply_qkv_tree(s["qkv"], s["qw"], s["kw"], s["cos"], s["sin"], s["k"], s["v"], s["seqlen"],
                                  s["parents"], num_heads=nq, num_kv_heads=nkv, head_dim=d, rotary_dim=c["rot"],
                                  interleaved=c["interleaved"], eps=EPS)
    return q, s["k"], s["v"]


def _own_attn(s):
    c = s["case"]
    return _kernels().tree_attention(s["q"], s["k"], s["v"], s["seqlen"], s["parents"],
                                     scale=HEADS[c["heads"]][2] ** -0.5, window=c["window"] or None)


def _own_verify(s):
    c = s["case"]
    return _kernels().verify_tree(s["logits"], s["tokens"], s["parents"], s["uniform"], temperature=c["temp"],
                                  top_p=c["top_p"], top_k=c["top_k"], draft_probs=s["probs"])


def _own_commit(s):
    n = _kernels().commit_tree(s["k"], s["v"], s["seqlen"], s["path"], s["accepted"])
    return n, s["k"], s["v"]


_own = {"qkv": _own_qkv, "attn": _own_attn, "verify": _own_verify, "commit": _own_commit}


def _tree(parents):
    """``reach [B, T, T]`` (1 where j is i or an ancestor of i), which nodes are present, and their depths."""
    t = parents.shape[1]
    i = torch.arange(t, device=parents.device)
    step = (parents.unsqueeze(-1) == i) & (parents < i).unsqueeze(-1)
    reach = step.float() + torch.eye(t, device=parents.device)
    for _ in range(6):  # paths of up to 2^6 steps
        reach = (reach @ reach > 0).float()
    present = (reach[:, :, 0] > 0) & (parents[:, :1] == -1)
    return reach, present, reach.sum(-1).long() - 1


def _rotate(x, cos, sin, rot, interleaved):
    """Rotary positions over the first ``rot`` of the last dimension; cos / sin ``[B, T, 1, rot]``."""
    h = rot // 2
    lo, hi = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :h], x[..., h:rot])
    a = lo * cos[..., :h] - hi * sin[..., :h]
    b = hi * cos[..., h:] + lo * sin[..., h:]
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_qkv(s):
    c = s["case"]
    nq, nkv, d = HEADS[c["heads"]]
    b, t, rot = c["batch"], c["nodes"], c["rot"]
    _, present, depth = _tree(s["parents"])
    pos = s["seqlen"].unsqueeze(1) + depth
    cos, sin = (s[n].float()[pos].unsqueeze(2) for n in ("cos", "sin"))
    x = s["qkv"].float().view(b, t, nq + 2 * nkv, d)
    norm = lambda y, w: y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w  # noqa: E731
    q = _rotate(norm(x[:, :, :nq], s["qw"]), cos, sin, rot, c["interleaved"])
    k = _rotate(norm(x[:, :, nq:nq + nkv], s["kw"]), cos, sin, rot, c["interleaved"])
    here = present.unsqueeze(-1).unsqueeze(-1)
    rows = torch.arange(b, device=DEV).unsqueeze(1)
    slot = s["seqlen"].unsqueeze(1) + torch.arange(t, device=DEV)
    for cache, new in ((s["k"], k), (s["v"], x[:, :, nq + nkv:])):
        cache[rows, :, slot] = torch.where(here, new.bfloat16(), cache[rows, :, slot])
    return torch.where(here, q, 0.0).bfloat16(), s["k"], s["v"]


def _plain_attn(s):
    c = s["case"]
    nq, nkv, d = HEADS[c["heads"]]
    b, t, n = c["batch"], c["nodes"], s["k"].shape[2]
    reach, present, depth = _tree(s["parents"])
    j = torch.arange(n, device=DEV)
    behind = j - s["seqlen"].unsqueeze(1)  # [B, n]: which node a slot holds, negative in the sequence
    node = behind.clamp(0, t - 1)
    # a slot's position: its index in the sequence, its node's depth behind it
    at = torch.where(behind < 0, j, s["seqlen"].unsqueeze(1) + torch.gather(depth, 1, node))
    seen = (behind < 0).unsqueeze(1) | ((behind >= 0) & (behind < t)).unsqueeze(1) & (
        torch.gather(reach, 2, node.unsqueeze(1).expand(b, t, n)) > 0)
    if c["window"]:
        seen = seen & (at.unsqueeze(1) > (s["seqlen"].unsqueeze(1) + depth).unsqueeze(-1) - c["window"])
    g = nq // nkv
    q = s["q"].float().view(b, t, nkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, nkv, t * g, d)
    x = (q @ s["k"].float().transpose(-1, -2)).view(b, nkv, t, g, n).mul_(d ** -0.5)
    x.masked_fill_(~seen.view(b, 1, t, 1, n), -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    y = (x.view(b, nkv, t * g, n) @ s["v"].float()).view(b, nkv, t, g, d) / total
    y = y.permute(0, 2, 1, 3, 4).reshape(b, t, nq, d)
    return torch.where(present.unsqueeze(-1).unsqueeze(-1), y, 0.0).bfloat16()


def _law(s):
    """The sampler's law at every node: ids and probabilities ``[B, T, k]``, most likely first, equal logits by id."""
    c = s["case"]
    x = s["logits"].float()
    bits = x.view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()  # sorts as the values do
    keys = order * 2 ** 32 + (2 ** 32 - 1 - torch.arange(c["vocab"], device=DEV))
    ids = 2 ** 32 - 1 - (torch.topk(keys, c["top_k"], dim=-1).values & (2 ** 32 - 1))
    z = torch.gather(x, 2, ids).double()
    p = torch.exp((z - z[..., :1]) / c["temp"])
    p = p / p.sum(-1, keepdim=True)
    p = torch.where(p.cumsum(-1) - p <= c["top_p"], p, 0.0)
    return ids, p / p.sum(-1, keepdim=True)


def _plain_verify(s):
    """In 64 bits, since a value next to a border decides a token."""
    c = s["case"]
    b, t = c["batch"], c["nodes"]
    ids, law = _law(s)
    _, present, _ = _tree(s["parents"])
    rows = torch.arange(b, device=DEV)
    u = s["uniform"].double()
    cur = torch.zeros(b, dtype=torch.long, device=DEV)
    count = torch.zeros(b, dtype=torch.long, device=DEV)
    path = torch.full((b, t + 1), -1, dtype=torch.long, device=DEV)
    path[:, 0] = 0
    p, support = law[:, 0], ids[:, 0]
    # a walk down the tree; a node's children follow it in index order, so one pass over the nodes takes every step
    for i in range(1, t):
        tried = present[:, i] & (s["parents"][:, i] == cur)
        token = s["tokens"][:, i:i + 1]
        is_it = support == token
        q = is_it.double() if s["probs"] is None else torch.gather(s["probs"][:, i], 1, support).double()
        qt = 1.0 if s["probs"] is None else torch.gather(s["probs"][:, i], 1, token).double().squeeze(1)
        took = tried & (u[:, i] * qt < torch.where(is_it, p, 0.0).sum(1))
        rest = (p - q).clamp(min=0.0)
        mass = rest.sum(1, keepdim=True)
        p = torch.where((tried & ~took).unsqueeze(1) & (mass > 0), rest / mass, p)
        p = torch.where(took.unsqueeze(1), law[:, i], p)
        support = torch.where(took.unsqueeze(1), ids[:, i], support)
        cur = torch.where(took, i, cur)
        count = count + took
        path.scatter_(1, torch.where(took, count, t).unsqueeze(1), i)
    path = torch.where(torch.arange(t, device=DEV) <= count.unsqueeze(1), path[:, :t], -1)
    cum = p.cumsum(1)
    pick = (cum <= u[:, :1] * cum[:, -1:]).sum(1).clamp(max=c["top_k"] - 1)
    drafted = torch.gather(s["tokens"], 1, path.clamp(min=0))
    out = torch.where(path >= 0, drafted, -1)[:, 1:]
    out = torch.cat([out, torch.full((b, 1), -1, dtype=torch.long, device=DEV)], 1)
    out[rows, count] = support[rows, pick]
    return out, count.int(), path.int()


def _plain_commit(s):
    c = s["case"]
    rows = torch.arange(c["batch"], device=DEV).unsqueeze(1)
    to = s["seqlen"].unsqueeze(1) + torch.arange(c["nodes"], device=DEV)
    come = torch.where(s["path"] >= 0, s["seqlen"].unsqueeze(1) + s["path"], to)
    for cache in s["k"] + s["v"]:
        cache[rows, :, to] = cache[rows, :, come]
    return s["seqlen"] + s["accepted"] + 1, s["k"], s["v"]


_plain = {"qkv": _plain_qkv, "attn": _plain_attn, "verify": _plain_verify, "commit": _plain_commit}


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------
def work(case):
    c = case
    b, t = c["batch"], c["nodes"]
    if c["kind"] == "verify":
        drafts = b * t * c["top_k"] * 4 if c["probs"] else 0
        return {"bytes": b * t * (c["vocab"] * 2 + 8 + 4 + 4 + 8 + 4) + drafts, "flops": b * t * c["vocab"]}
    nq, nkv, d = HEADS[c["heads"]]
    mean = lambda n: n if b == 1 else (n + 0.75 * n * (b - 1)) / b  # noqa: E731  (a row has half of n to n)
    nodes, length = mean(t), mean(c["length"])
    if c["kind"] == "qkv":
        return {"bytes": b * nodes * ((nq + 2 * nkv) * d * 4 + c["rot"] * 4), "flops": b * nodes * (nq + nkv) * d * 10}
    if c["kind"] == "commit":
        moved = max(1.0, math.log2(t) / 2)
        return {"bytes": 2 * c["layers"] * b * nkv * d * moved * 4 + b * t * 4, "flops": 0}
    span = min(length, c["window"]) if c["window"] else length
    return {"bytes": b * ((span + nodes) * 2 * nkv * d * 2 + 2 * nodes * nq * d * 2),
            "flops": 4 * b * nodes * nq * d * span}


# ---------------------------------------------------------------------------
# The same values in 64 bits, node by node.
# ---------------------------------------------------------------------------
def _branches(parents):
    """Per row and node the list of nodes from the root to it, None for padding."""
    rows = []
    for p in parents.tolist():
        line = [[0] if p[0] == -1 else None]
        for i in range(1, len(p)):
            up = line[p[i]] if 0 <= p[i] < i else None
            line.append(None if up is None else up + [i])
        rows.append(line)
    return rows


def exact(case, seed):
    if case["kind"] == "commit":
        return None  # copies: nothing is computed
    s = prepare(case, seed)
    return {"qkv": _exact_qkv, "attn": _exact_attn, "verify": _exact_verify}[case["kind"]](s, case)


def _exact_qkv(s, c):
    nq, nkv, d = HEADS[c["heads"]]
    rot, half = c["rot"], c["rot"] // 2
    out = torch.zeros(c["batch"], c["nodes"], nq, d, dtype=torch.float64, device=DEV)
    k, v = s["k"].double(), s["v"].double()
    dims = torch.arange(rot, device=DEV)
    if c["interleaved"]:
        other, col, sign = dims ^ 1, dims // 2 + (dims % 2) * half, (dims % 2) * 2.0 - 1.0
    else:
        other, col = (dims + half) % rot, dims
        sign = torch.where(dims < half, -1.0, 1.0)
    weights = torch.cat([s["qw"].double().expand(nq, d), s["kw"].double().expand(nkv, d)])
    for b, line in enumerate(_branches(s["parents"])):
        n = int(s["seqlen"][b])
        for i, up in enumerate(line):
            if up is None:
                continue
            x = s["qkv"][b, i].double().view(nq + 2 * nkv, d)
            y = x[:nq + nkv]
            y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * weights
            co, si = (s[w][n + len(up) - 1].double()[col] for w in ("cos", "sin"))
            y[:, :rot] = y[:, dims] * co + sign * y[:, other] * si
            out[b, i] = y[:nq]
            k[b, :, n + i], v[b, :, n + i] = y[nq:], x[nq + nkv:]
    return out, k, v


def _exact_attn(s, c):
    nq, nkv, d = HEADS[c["heads"]]
    b, t = c["batch"], c["nodes"]
    out = torch.zeros(b, t, nq, d, dtype=torch.float64, device=DEV)
    for r, line in enumerate(_branches(s["parents"])):
        n = int(s["seqlen"][r])
        here = [i for i, up in enumerate(line) if up is not None]
        on = torch.zeros(t, n + t, dtype=torch.bool)
        for i in here:
            pos = n + len(line[i]) - 1
            lo = max(0, pos + 1 - c["window"]) if c["window"] else 0
            on[i, lo:n] = True
            for dist, a in enumerate(reversed(line[i])):
                on[i, n + a] = not c["window"] or dist < c["window"]
        on = on[here].to(DEV)
        k, v = (s[w][r, :, :n + t].double() for w in ("k", "v"))
        for h in range(nq):
            x = s["q"][r, here, h].double() @ k[h * nkv // nq].t() * d ** -0.5
            p = torch.softmax(torch.where(on, x, -math.inf), -1)
            out[r, here, h] = p @ v[h * nkv // nq]
    return out


def _exact_verify(s, c):
    b, t = c["batch"], c["nodes"]
    logits = s["logits"]
    tokens, u, parents = (s[w].cpu().numpy() for w in ("tokens", "uniform", "parents"))
    out, count, path = np.full((b, t), -1), np.zeros(b, np.int64), np.full((b, t), -1)

    def law(r, i):
        z = logits[r, i].double().cpu().numpy()
        top = np.argsort(-z, kind="stable")[:c["top_k"]]
        p = np.exp((z[top] - z[top[0]]) / c["temp"])
        p /= p.sum()
        p[np.concatenate([[0.0], np.cumsum(p)[:-1]]) > c["top_p"]] = 0.0
        return list(top), p / p.sum()

    for r, line in enumerate(_branches(s["parents"])):
        path[r, 0], cur, (ids, p) = 0, 0, law(r, 0)
        while True:
            for i in range(cur + 1, t):
                if line[i] is None or parents[r, i] != cur:
                    continue
                tok = int(tokens[r, i])
                if s["probs"] is None:
                    qt, q = 1.0, np.array([float(k == tok) for k in ids])
                else:
                    row = s["probs"][r, i].double().cpu().numpy()
                    qt, q = row[tok], row[ids]
                if float(u[r, i]) * qt < (p[ids.index(tok)] if tok in ids else 0.0):
                    out[r, count[r]] = tok
                    count[r] += 1
                    path[r, count[r]], cur, (ids, p) = i, i, law(r, i)
                    break
                rest = np.maximum(p - q, 0.0)
                if rest.sum() > 0:
                    p = rest / rest.sum()
            else:
                break
        cum = np.cumsum(p)
        out[r, count[r]] = ids[min(int((cum <= float(u[r, 0]) * cum[-1]).sum()), c["top_k"] - 1)]
    return torch.from_numpy(out), torch.from_numpy(count).int(), torch.from_numpy(path).int()
