"""Operators around a KV cache at the sizes they are used at: appending projected tokens (norms, rotary positions),
attention for a tree of drafted tokens, decode that accumulates each key's attention weight, and the eviction that
those weights decide.

The cache is k, v [batch][kv_heads][k_stride][dim] in 16 bits with kv_len [batch] int32 on the device.  `run` computes
an operator in elementary torch operations (`own` false) or calls this repository's kernels (`own` true).
"""
import math
import sys

import numpy as np
import torch

own = False

HALVES, PAIRS = 1, 2  # rotation partners: (i, i + rot / 2) or (2i, 2i + 1)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # one token of each of 8 sequences between two decode steps: launch latency
        dict(name="append_token", op="append", dtype="bf16", batch=8, n_tok=1, ragged=False, lo=1024, hi=4095, far=0,
             heads=32, kv_heads=8, dim=128, rot=128, layout=HALVES, norm=True, gated=False),
        # drafted tokens with gated 256-wide heads, a quarter rotated in adjacent pairs, at positions near a million
        # (a cache whose early tokens were evicted), ragged drafts
        dict(name="append_draft_d256", op="append", dtype="fp16", batch=8, n_tok=37, ragged=True, lo=1000, hi=4000,
             far=1000000, heads=16, kv_heads=2, dim=256, rot=64, layout=PAIRS, norm=True, gated=True),
        # two prompts of 8192 tokens into an empty cache
        dict(name="append_prompt", op="append", dtype="bf16", batch=2, n_tok=8192, ragged=False, lo=0, hi=0, far=0,
             heads=32, kv_heads=8, dim=128, rot=128, layout=HALVES, norm=True, gated=False),
        # one request of a short context, 8 drafted tokens: latency
        dict(name="tree_short", op="tree", dtype="fp16", batch=1, n_tok=8, ragged=False, lo=512, hi=512, heads=16,
             kv_heads=8, dim=128),
        # a batch of long contexts, 16 drafted tokens each: the cache read is all
        dict(name="tree_16", op="tree", dtype="bf16", batch=8, n_tok=16, ragged=False, lo=16384, hi=32768, heads=32,
             kv_heads=8, dim=128),
        # the same with 64-token trees: 256 query rows share a key
        dict(name="tree_64", op="tree", dtype="bf16", batch=8, n_tok=64, ragged=False, lo=16384, hi=32768, heads=32,
             kv_heads=8, dim=128),
        # 256-wide heads, odd trees, ragged drafts and lengths
        dict(name="tree_37_d256", op="tree", dtype="fp16", batch=4, n_tok=37, ragged=True, lo=1001, hi=9001, heads=16,
             kv_heads=2, dim=256),
        # a short context of 64-wide heads, one kv head a query head: latency
        dict(name="weights_short", op="weights", dtype="bf16", batch=1, lo=777, hi=777, heads=8, kv_heads=8, dim=64),
        # batched decode over long contexts, weights kept for a later eviction
        dict(name="weights_batch", op="weights", dtype="fp16", batch=8, lo=16384, hi=32768, heads=32, kv_heads=8,
             dim=128),
        # one very long sequence of 256-wide heads
        dict(name="weights_long_d256", op="weights", dtype="bf16", batch=1, lo=131072, hi=131072, heads=16,
             kv_heads=2, dim=256),
        # two short caches cut to half
        dict(name="evict_short_d256", op="evict", dtype="fp16", batch=2, lo=701, hi=1301, kv_heads=2, dim=256, sinks=4,
             recent=64, budget=512),
        # a batch of prompts' caches compressed into small decode caches
        dict(name="evict_prompts", op="evict", dtype="bf16", batch=8, lo=16384, hi=32768, kv_heads=8, dim=128, sinks=4,
             recent=256, budget=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "tree", "weights", "evict"])
    dtype, dim = rng.choice(["fp16", "bf16"]), rng.choice([64, 128, 256])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8])
    batch = _log(rng, 1, 16)
    c = dict(op=op, dtype=dtype, batch=batch, dim=dim, kv_heads=kv_heads)
    # keys of the longest sequence: the cache stays within that of the largest listed case
    top = min(65536, (1 << 28) // (batch * kv_heads * dim))
    if op == "append":
        n_tok = _log(rng, 1, max(2, min(8192, (1 << 26) // (batch * kv_heads * (group + 2) * dim))))
        lo = _log(rng, 1, 4096) - 1
        return dict(c, n_tok=n_tok, ragged=rng.random() < 0.5, lo=lo, hi=lo + rng.randrange(512),
                    far=rng.choice([0, 0, 100000, 1000000]), heads=kv_heads * group,
                    rot=rng.choice([dim, dim // 2, dim // 4, dim - 2]), layout=rng.choice([HALVES, PAIRS]),
                    norm=rng.random() < 0.7, gated=rng.random() < 0.3)
    if op == "tree":
        n_tok = _log(rng, 1, 100)
        top = max(256, min(top, (1 << 29) // (batch * kv_heads * group * n_tok)))
        hi = _log(rng, 64, top)
        return dict(c, n_tok=n_tok, ragged=rng.random() < 0.5, lo=rng.randrange(hi + 1), hi=hi,
                    heads=kv_heads * group)
    hi = _log(rng, 64, top)
    lo = rng.randrange(1, hi + 1)
    if op == "weights":
        return dict(c, lo=lo, hi=hi, heads=kv_heads * group)
    budget = rng.randrange(32, max(33, min(8192, hi)))
    recent = rng.randrange(budget // 2 + 1)
    return dict(c, lo=lo, hi=hi, sinks=rng.randrange(min(9, budget - recent)), recent=recent, budget=budget)


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _freqs(rot):
    """Radians a position of each rotated pair, for a context extended 4 times by parts: pairs that turn less than
    once over the 8192 positions of training are slowed 4 times, those that turn over 32 times are kept."""
    i = np.arange(rot // 2, dtype=np.float64)
    f = 500000.0 ** (-2.0 * i / max(rot, 1))
    keep = np.clip((8192.0 * f / (2.0 * math.pi) - 1.0) / 31.0, 0.0, 1.0)
    return f * (keep + (1.0 - keep) / 4.0)


def _tree(rs, batch, n):
    """Visibility words [batch][n][ceil(n / 32)]: a token sees itself and its ancestors; a parent is one of the few
    tokens before it, or the last cached one."""
    see = np.zeros((batch, n, n), bool)
    who = np.arange(batch)
    for i in range(n):
        parent = i - 1 - rs.integers(0, 6, batch)
        has = parent >= 0
        see[who[has], i] = see[who[has], parent[has]]
        see[:, i, i] = True
    words = (n + 31) // 32
    bits = np.zeros((batch, n, words * 32), np.uint64)
    bits[:, :, :n] = see
    w = (bits.reshape(batch, n, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1)
    return see, torch.from_numpy(w.astype(np.uint32).view(np.int32))


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rs = np.random.default_rng(seed)
    dt, B, KV, D = DTYPES[c["dtype"]], c["batch"], c["kv_heads"], c["dim"]
    n = c.get("n_tok", 0)
    S = (c["hi"] + max(n, 1) + 63) // 64 * 64
    lens = rs.integers(c["lo"], c["hi"] + 1, B).astype(np.int32)
    s = dict(c, S=S, dt=dt, kv_len=torch.from_numpy(lens).cuda(), lens=lens)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    # a cache in use: rows of unit variance, as the producers' norms leave them
    s["k"], s["v"] = randn(B, KV, S, D, dtype=dt), randn(B, KV, S, D, dtype=dt)
    if n:
        new = rs.integers(1, n + 1, B) if c["ragged"] else np.full(B, n)
        s["n_new"] = torch.from_numpy(new.astype(np.int32)).cuda() if c["ragged"] else None
    if c["op"] == "append":
        H = c["heads"]
        s["q_stride"] = 2 * D if c["gated"] else D
        s["k_col0"] = H * s["q_stride"]
        s["v_col0"] = s["k_col0"] + KV * D
        s["ld"] = s["v_col0"] + KV * D
        s["x"] = 3.0 * randn(B * n, s["ld"])
        first = lens.astype(np.int64) + (rs.integers(c["far"], c["far"] + 1000, B) if c["far"] else 0)
        pos = first[:, None] + np.arange(n)
        s["pos"] = torch.from_numpy(pos.astype(np.int32)).cuda() if c["far"] else None
        s["freq"] = torch.from_numpy(_freqs(c["rot"])).cuda()
        s["amplitude"] = 0.1 * math.log(4.0) + 1.0
        s["wq"] = 1.0 + 0.1 * randn(D) if c["norm"] else None
        s["wk"] = 1.0 + 0.1 * randn(D) if c["norm"] else None
        s["q"] = torch.zeros(B, n, H, D, dtype=dt, device="cuda")
    elif c["op"] == "tree":
        s["q"] = randn(B, n, c["heads"], D, dtype=dt)
        s["see"], mask = _tree(rs, B, n)
        s["mask"] = mask.cuda()
        s["o"] = torch.zeros(B, n, c["heads"] * D, dtype=dt, device="cuda")
    elif c["op"] == "weights":
        s["q"] = randn(B, c["heads"], D, dtype=dt)
        s["weight"] = torch.rand(B, KV, S, generator=g, device="cuda")
        s["o"] = torch.zeros(B, c["heads"] * D, dtype=dt, device="cuda")
    else:
        # heavy-tailed sums, on a grid so that ties occur
        s["weight"] = torch.round(torch.exp(2.0 * randn(B, KV, S)) * 1024.0) / 1024.0
        bud = c["budget"]
        s["k_out"] = torch.zeros(B, KV, bud, D, dtype=dt, device="cuda")
        s["v_out"], s["weight_out"] = torch.zeros_like(s["k_out"]), torch.zeros(B, KV, bud, device="cuda")
        s["kept"] = torch.zeros(B, KV, bud, dtype=torch.int32, device="cuda")
        s["new_len"] = torch.zeros(B, dtype=torch.int32, device="cuda")
    return s


# ---- the framework's kernels ----------------------------------------------------------------------------------------

_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        if "mako-common_b200" not in sys.path:
            sys.path.insert(0, "mako-common_b200")
        import mako_attn
        _ctx = mako_attn.Context(torch.cuda.current_device())
        _ctx.set_option(mako_attn.OPT_OUTPUT_16BIT, 1)
    return _ctx


def _own(s):
    ctx = _context()
    if s["op"] == "append":
        ctx.cache_append(s["x"], s["ld"], 0, s["q_stride"], s["k_col0"], s["v_col0"], s["batch"], s["n_tok"],
                         s["n_new"], s["kv_len"], s["pos"], s["heads"], s["kv_heads"], s["dim"], s["rot"], s["layout"],
                         s["freq"], s["amplitude"], s["wq"], s["wk"], EPS, s["q"], s["k"], s["v"], s["S"])
        return [s["q"], s["k"], s["v"]]
    if s["op"] == "tree":
        ctx.attention_tree(s["q"], s["k"], s["v"], s["o"], s["batch"], s["n_tok"], s["n_new"], s["kv_len"], s["hi"],
                           s["heads"], s["kv_heads"], s["dim"], s["S"], s["mask"])
        return [s["o"]]
    if s["op"] == "weights":
        ctx.attention_decode_weights(s["q"], s["k"], s["v"], s["o"], s["weight"], s["kv_len"], s["hi"], s["heads"],
                                     s["kv_heads"], s["dim"], s["S"])
        return [s["o"], s["weight"]]
    ctx.cache_evict(s["k"], s["v"], s["weight"], s["kv_len"], s["hi"], s["kv_heads"], s["dim"], s["S"], s["sinks"],
                    s["recent"], s["budget"], s["k_out"], s["v_out"], s["weight_out"], s["budget"], s["kept"],
                    s["new_len"])
    return [s["k_out"], s["v_out"], s["weight_out"], s["kept"], s["new_len"]]


# ---- plain forms ----------------------------------------------------------------------------------------------------


def _live(s):
    """[batch][n_tok]: the tokens that there are."""
    i = torch.arange(s["n_tok"], device="cuda")[None]
    return i < (s["n_new"][:, None] if s["n_new"] is not None else s["n_tok"])


def _norm(u, w):
    return u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * w if w is not None else u


def _rotate(u, cos, sin, rot, layout):
    """u [batch][n_tok][heads][dim]; cos, sin [batch][n_tok][1][rot / 2]."""
    r, rest = u[..., :rot], u[..., rot:]
    if layout == HALVES:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = r[..., 0::2], r[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _append(s):
    B, n, H, KV, D, rot = s["batch"], s["n_tok"], s["heads"], s["kv_heads"], s["dim"], s["rot"]
    x = s["x"].view(B, n, s["ld"])
    q = x[..., :s["k_col0"]].view(B, n, H, s["q_stride"])[..., :D]
    k = x[..., s["k_col0"]:s["v_col0"]].view(B, n, KV, D)
    v = x[..., s["v_col0"]:].view(B, n, KV, D)
    row = s["kv_len"][:, None].long() + torch.arange(n, device="cuda")
    angle = (s["pos"] if s["pos"] is not None else row).double()[..., None] * s["freq"]
    cos = (torch.cos(angle) * s["amplitude"]).float()[:, :, None]
    sin = (torch.sin(angle) * s["amplitude"]).float()[:, :, None]
    q = _rotate(_norm(q, s["wq"]), cos, sin, rot, s["layout"])
    k = _rotate(_norm(k, s["wk"]), cos, sin, rot, s["layout"])
    live = _live(s)
    s["q"].copy_(torch.where(live[..., None, None], q.to(s["dt"]), s["q"]))
    at = row[:, None, :, None].expand(B, KV, n, D)
    for name, new in (("k", k), ("v", v)):
        old = s[name].gather(2, at)
        s[name].scatter_(2, at, torch.where(live[:, None, :, None], new.to(s["dt"]).transpose(1, 2), old))
    return [s["q"], s["k"], s["v"]]


def _softmax(score, see):
    """Weights over the last axis of what is seen, 0 where nothing is."""
    score = score.masked_fill_(~see, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total > 0, total, 1.0))


def _attend(s, q, see):
    """q [batch][n][heads][dim], see [batch][n][keys]: the output rows and the weights [batch][kv][group * n][keys]."""
    B, n, H, D = q.shape
    KV, L = s["kv_heads"], see.shape[-1]
    G = H // KV
    rows = q.float().view(B, n, KV, G, D).permute(0, 2, 3, 1, 4).reshape(B, KV, G * n, D)
    k, v = s["k"][:, :, :L].float(), s["v"][:, :, :L].float()
    score = (rows @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(D)).view(B, KV, G, n, L)
    p = _softmax(score, see[:, None, None]).view(B, KV, G * n, L)
    o = (p @ v).view(B, KV, G, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, H * D)
    return o, p


def _attend_tree(s):
    B, n, L = s["batch"], s["n_tok"], s["hi"] + s["n_tok"]
    bits = (s["mask"][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    bits = bits.flatten(-2)[..., :n].bool()  # [batch][token][drafted]
    j, length = torch.arange(L, device="cuda"), s["kv_len"][:, None]
    drafted = j - length  # [batch][keys]
    live = _live(s)
    seen = (bits & live[:, None]).gather(2, drafted.clamp(0, n - 1)[:, None].expand(B, n, L).long())
    see = (j < length)[:, None] | (seen & ((drafted >= 0) & (drafted < n))[:, None])
    o, _ = _attend(s, s["q"], see)
    s["o"].copy_(torch.where(live[..., None], o.to(s["dt"]), s["o"]))
    return [s["o"]]


def _weights(s):
    j = torch.arange(s["hi"], device="cuda")
    o, p = _attend(s, s["q"][:, None], (j < s["kv_len"][:, None])[:, None])
    s["o"].copy_(o[:, 0].to(s["dt"]))
    s["weight"][..., :s["hi"]] += p.sum(2)
    return [s["o"], s["weight"]]


def _evict(s):
    B, KV, D, bud = s["batch"], s["kv_heads"], s["dim"], s["budget"]
    j, length = torch.arange(s["S"], device="cuda"), s["kv_len"][:, None, None]
    must = (j < s["sinks"]) | (j >= length - s["recent"])
    score = s["weight"].masked_fill(must, math.inf).masked_fill(j >= length, -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :bud]
    new_len = length.clamp(max=bud)
    kept = torch.arange(bud, device="cuda") < new_len  # [batch][1][budget]
    pad = bud - best.shape[-1]
    best = torch.cat([best, best.new_zeros(B, KV, pad)], -1) if pad > 0 else best
    at = torch.sort(best.masked_fill(~kept, s["S"]), dim=-1).values
    rows = at.clamp(max=s["S"] - 1)
    wide = rows[..., None].expand(B, KV, bud, D)
    for name, out in (("k", "k_out"), ("v", "v_out")):
        s[out].copy_(torch.where(kept[..., None], s[name].gather(2, wide), s[out]))
    s["weight_out"].copy_(torch.where(kept, s["weight"].gather(2, rows), s["weight_out"]))
    s["kept"].copy_(torch.where(kept, at, -1))
    s["new_len"].copy_(new_len.view(B))
    return [s["k_out"], s["v_out"], s["weight_out"], s["kept"], s["new_len"]]


def run(state):
    if own:
        return _own(state)
    return {"append": _append, "tree": _attend_tree, "weights": _weights, "evict": _evict}[state["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------


def work(case):
    c = case
    B, KV, D = c["batch"], c["kv_heads"], c["dim"]
    mean = (c["lo"] + c["hi"]) / 2
    if c["op"] == "append":
        tokens = B * ((c["n_tok"] + 1) / 2 if c["ragged"] else c["n_tok"])
        values = tokens * (c["heads"] + 2 * KV) * D
        return {"bytes": values * 6, "flops": values * 8}
    if c["op"] == "tree":
        new = (c["n_tok"] + 1) / 2 if c["ragged"] else c["n_tok"]
        keys = B * KV * (mean + new)
        return {"bytes": keys * D * 4 + B * new * c["heads"] * D * 4,
                "flops": 4.0 * D * keys * new * c["heads"] / KV}
    if c["op"] == "weights":
        keys = B * KV * mean
        return {"bytes": keys * (D * 4 + 8) + B * c["heads"] * D * 4, "flops": 4.0 * D * keys * c["heads"] / KV}
    rows = B * KV * min(mean, c["budget"])
    return {"bytes": B * KV * mean * 4 + rows * (D * 8 + 8), "flops": B * KV * mean}


# ---- 64 bits --------------------------------------------------------------------------------------------------------


def _exact_append(s):
    B, n, H, KV, D, rot = s["batch"], s["n_tok"], s["heads"], s["kv_heads"], s["dim"], s["rot"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    x = s["x"].double().view(B, n, s["ld"])
    half = rot // 2
    pair = np.arange(half)
    first = pair if s["layout"] == HALVES else 2 * pair
    second = pair + half if s["layout"] == HALVES else 2 * pair + 1
    for b in range(B):
        m, l = (int(s["n_new"][b]) if s["n_new"] is not None else n), int(s["lens"][b])
        at = s["pos"][b, :m].double() if s["pos"] is not None else l + torch.arange(m, device="cuda").double()
        turn = torch.polar(torch.full((m, 1, half), s["amplitude"], device="cuda", dtype=torch.float64),
                           (at[:, None] * s["freq"][None])[:, None])

        def head(col0, step, count, w, rotate=True):
            cols = col0 + step * np.arange(count)[:, None] + np.arange(D)
            u = x[b, :m][:, torch.from_numpy(cols).cuda()]
            if w is not None:
                u = u / (u.square().sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
            if rotate and rot:
                z = torch.complex(u[..., first], u[..., second]) * turn
                u[..., first], u[..., second] = z.real, z.imag
            return u

        q[b, :m] = head(0, s["q_stride"], H, s["wq"])
        k[b, :, l:l + m] = head(s["k_col0"], D, KV, s["wk"]).transpose(0, 1)
        v[b, :, l:l + m] = head(s["v_col0"], D, KV, None, False).transpose(0, 1)
    return [q, k, v]


def _exact_rows(q, k, v, see):
    """q [rows][dim], k, v [keys][dim], see [rows][keys]: the output rows and weights."""
    z = (q @ k.T / math.sqrt(q.shape[-1])).masked_fill(~see, -math.inf)
    p = torch.nan_to_num(torch.softmax(z, -1))
    return p @ v, p


def _exact_attention(s):
    tree = s["op"] == "tree"
    o, H, KV, D = s["o"].double(), s["heads"], s["kv_heads"], s["dim"]
    w = None if tree else s["weight"].double()
    q = s["q"].double() if tree else s["q"].double()[:, None]
    for b in range(s["batch"]):
        l, m = int(s["lens"][b]), 1
        see = np.ones((1, l), bool)
        if tree:
            m = int(s["n_new"][b]) if s["n_new"] is not None else s["n_tok"]
            see = np.concatenate([np.ones((m, l), bool), s["see"][b, :m, :m]], 1)
        see = torch.from_numpy(see).cuda()
        for h in range(H):
            kv = h // (H // KV)
            k, v = s["k"][b, kv, :see.shape[1]].double(), s["v"][b, kv, :see.shape[1]].double()
            r, p = _exact_rows(q[b, :m, h], k, v, see)
            if tree:
                o[b, :m, h * D:(h + 1) * D] = r
            else:
                o[b, h * D:(h + 1) * D] = r[0]
                w[b, kv, :l] += p[0]
    return [o] if tree else [o, w]


def _exact_evict(s):
    k, v, w = s["k_out"].double(), s["v_out"].double(), s["weight_out"].double()
    kept = np.full(tuple(s["kept"].shape), -1, np.int32)
    weight = s["weight"].cpu().numpy().astype(np.float64)
    for b in range(s["batch"]):
        l = int(s["lens"][b])
        lo, hi = min(s["sinks"], l), max(l - s["recent"], 0)
        for h in range(s["kv_heads"]):
            if l <= s["budget"]:
                rows = np.arange(l)
            else:
                middle = np.arange(lo, hi)
                order = np.lexsort((middle, -weight[b, h, lo:hi]))
                top = middle[order[:s["budget"] - lo - (l - hi)]]
                rows = np.sort(np.concatenate([np.arange(lo), top, np.arange(hi, l)]))
            kept[b, h, :len(rows)] = rows
            at = torch.from_numpy(rows).cuda()
            k[b, h, :len(rows)], v[b, h, :len(rows)] = s["k"][b, h, at].double(), s["v"][b, h, at].double()
            w[b, h, :len(rows)] = s["weight"][b, h, at].double()
    return [k, v, w, torch.from_numpy(kept), torch.from_numpy(np.minimum(s["lens"], s["budget"]))]


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "evict": _exact_evict}.get(s["op"], _exact_attention)(s)
