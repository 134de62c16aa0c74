"""Cases of the operators for trees of drafted tokens over a paged cache, for measurement and comparison.

A serving step with drafted trees runs five operators, one after another:

- append: the new tokens (a tree's nodes, each below an earlier one) are rotated by
  their depth in the tree; keys and values go to consecutive slots of their pages;
- attend: each new token attends to its sequence's context and, among the new ones, to
  those that its row of a bit mask names (its ancestors and itself);
- sample: logits to tokens by temperature, top-k, top-p and min-p, row by row, from
  given random numbers, with the probabilities where they are asked for;
- accept: the way down the tree, as long as the token sampled at a node is a child's;
- keep: the accepted nodes' keys and values move to the slots behind the context, in every
  layer.

`own` False: the operators in plain torch operations. `own` True: the library's calls.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one user's tree: the call's latency (TinyLlama heads, the f16 cache under f32 activations)
        {"name": "append one tree", "op": "append", "seqs": 1, "q_min": 26, "q_max": 26, "kv_min": 333, "kv_max": 333, "heads": 32,
         "kv_heads": 4, "dim": 64, "rot": 64, "halves": False, "norms": False, "theta": 10000.0, "act": "f32", "cache": "f16", "page": 16, "by_head": True, "mix": 1},
        # a batch of trees far into their sequences, norms of queries and keys, 70B heads
        {"name": "append trees", "op": "append", "seqs": 64, "q_min": 17, "q_max": 64, "kv_min": 65, "kv_max": 4096, "heads": 64,
         "kv_heads": 8, "dim": 128, "rot": 128, "halves": True, "norms": True, "theta": 500000.0, "act": "bf16", "cache": "bf16", "page": 16, "by_head": False, "mix": 2},
        # one user's tree over a short chat: latency
        {"name": "attend one tree", "op": "attend", "seqs": 1, "q_min": 26, "q_max": 26, "kv_min": 333, "kv_max": 333, "heads": 32,
         "kv_heads": 4, "dim": 64, "act": "f32", "cache": "f16", "page": 16, "by_head": True, "window": 0, "mix": 3},
        # a serving batch of trees of many sizes, ragged lengths, 70B heads
        {"name": "attend trees", "op": "attend", "seqs": 32, "q_min": 1, "q_max": 64, "kv_min": 65, "kv_max": 4096, "heads": 64,
         "kv_heads": 8, "dim": 128, "act": "bf16", "cache": "bf16", "page": 16, "by_head": False, "window": 0, "mix": 4},
        # trees and single tokens in one batch, a sliding window, the f32 cache of the reference's numerics, TinyLlama heads
        {"name": "attend window f32", "op": "attend", "seqs": 9, "q_min": 1, "q_max": 48, "kv_min": 49, "kv_max": 1500, "heads": 32,
         "kv_heads": 4, "dim": 64, "act": "f32", "cache": "f32", "page": 16, "by_head": True, "window": 511, "mix": 5},
        # one user's token by the framework's default settings: latency
        {"name": "sample one", "op": "sample", "rows": 1, "vocab": 32000, "act": "f32", "spread": 2.5, "params": "default", "probs": False, "mix": 6},
        # a token for every node of a batch of trees, requests of many settings, 16-bit logits
        {"name": "sample trees", "op": "sample", "rows": 416, "vocab": 32000, "act": "bf16", "spread": 2.5, "params": "mixed", "probs": False, "mix": 7},
        # a large batch over a large vocabulary of odd size, with the probabilities that a draft's verification reads
        {"name": "sample with probabilities", "op": "sample", "rows": 192, "vocab": 100003, "act": "f32", "spread": 3.0, "params": "mixed", "probs": True, "mix": 8},
        # one user's tree: latency
        {"name": "accept one", "op": "accept", "seqs": 1, "q_min": 26, "q_max": 26, "vocab": 32000, "mix": 9},
        # a large batch of large trees
        {"name": "accept batch", "op": "accept", "seqs": 256, "q_min": 32, "q_max": 128, "vocab": 32000, "mix": 10},
        # one user's accepted tokens, 22 layers: latency
        {"name": "keep one", "op": "keep", "seqs": 1, "q_min": 26, "q_max": 26, "kv_min": 333, "kv_max": 333, "kept": 5, "layers": 22, "kv_heads": 4,
         "dim": 64, "cache": "f16", "page": 16, "by_head": True, "mix": 11},
        # a serving batch's, 80 layers
        {"name": "keep batch", "op": "keep", "seqs": 32, "q_min": 32, "q_max": 64, "kv_min": 65, "kv_max": 200, "kept": 8, "layers": 80, "kv_heads": 8,
         "dim": 128, "cache": "bf16", "page": 16, "by_head": False, "mix": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample", "sample", "accept", "keep"])
    mix = rng.randrange(1 << 30)
    if op == "sample":
        vocab = _spread(rng, 1000, 131072)
        return {"op": op, "rows": _spread(rng, 1, max(1, min(512, 19_000_000 // vocab))), "vocab": vocab, "act": rng.choice(["f32", "f16", "bf16"]),
                "spread": rng.choice([1.0, 2.5, 4.0]), "params": rng.choice(["default", "mixed", "mixed", "top_p", "none"]), "probs": rng.random() < 0.4, "mix": mix}
    if op == "accept":
        q_max = _spread(rng, 1, 160)
        return {"op": op, "seqs": _spread(rng, 1, 256), "q_min": rng.randint(1, q_max), "q_max": q_max, "vocab": _spread(rng, 1000, 131072), "mix": mix}
    heads, kv_heads, dim = rng.choice([(32, 4, 64), (32, 32, 128), (64, 8, 128), (8, 2, 64), (15, 5, 64), (8, 1, 128)])
    act, cache = rng.choice([("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "bf16")])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    case = {"op": op, "kv_heads": kv_heads, "dim": dim, "cache": cache, "page": page, "by_head": rng.random() < 0.5, "mix": mix}
    if op == "keep":
        case["layers"] = _spread(rng, 1, 80)
        case["q_max"] = _spread(rng, 2, 96)
        case["kept"] = rng.randint(1, min(12, case["q_max"]))
        case["q_min"] = rng.randint(1, case["q_max"])
        # the pools of all layers are at hand
        per_seq = case["layers"] * kv_heads * dim * (case["q_max"] + 60 + page)
        case["seqs"] = _spread(rng, 1, max(1, min(64, 300_000_000 // per_seq)))
        case["kv_min"], case["kv_max"] = case["q_max"], case["q_max"] + rng.randint(0, 60)
        return case
    case.update(heads=heads, act=act)
    case["seqs"] = _spread(rng, 1, 48)
    case["q_max"] = _spread(rng, 1, 160 if op == "append" else 128)
    case["q_min"] = 1 if rng.random() < 0.7 else case["q_max"]
    if op == "append":
        case["seqs"] = max(1, min(case["seqs"], 2500 // case["q_max"]))
        case["kv_max"] = case["q_max"] + _spread(rng, 1, 2000)
        case["kv_min"] = case["q_max"]
        case.update(rot=dim if rng.random() < 0.7 else dim // 2, halves=rng.random() < 0.5, norms=rng.random() < 0.5, theta=rng.choice([10000.0, 500000.0]))
    else:
        # the plain form holds seqs x largest tree x longest sequence x heads scores, and its sequences' keys in 32 bits
        most = min(500_000_000 // (case["seqs"] * case["q_max"] * heads), (39 if cache == "f32" else 78) * 1_000_000 // (case["seqs"] * kv_heads * dim), 60000)
        case["kv_max"] = max(case["q_max"], _spread(rng, 1, max(2, most)))
        case["kv_min"] = max(1, case["kv_max"] // 8)
        case["window"] = 0 if rng.random() < 0.7 else _spread(rng, 1, max(2, case["kv_max"]))
    return case


def _lengths(case):
    """New tokens and cached tokens (new ones included) of each sequence: by the case alone."""
    r = random.Random(case["mix"])
    q = [r.randint(case["q_min"], case["q_max"]) for _ in range(case["seqs"])]
    kv = [max(n, r.randint(case.get("kv_min", 1), case.get("kv_max", 1))) for n in q]
    q[0] = case["q_max"]
    kv[0] = max(q[0], case.get("kv_max", 1))
    return q, kv


def _trees(case, q_len, seed):
    """Each new token's parent (among its sequence's new tokens; -1: the root), its depth, its ancestors and itself as
    bits of 32-bit words."""
    r = random.Random(case["mix"] * 1000003 + seed)
    words = -(-max(q_len) // 32)
    parent, depth, mask = [], [], []
    for n in q_len:
        p, d, m = [-1], [0], [1]
        for i in range(1, n):
            up = i - 1 if r.random() < 0.3 else r.randrange(max(0, i - 12), i)  # chains, and branches near the end
            p.append(up)
            d.append(d[up] + 1)
            m.append(m[up] | 1 << i)
        parent += p
        depth += d
        mask += [[(x >> 32 * w) & 0xffffffff for w in range(words)] for x in m]
    mask = torch.tensor(mask, dtype=torch.int64)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).int()
    return parent, depth, mask, words


def _ways(case, q_len):
    """The accepted nodes of each tree: its first branch held for a while, then a later one did (chains come before
    side branches). By the case alone."""
    r = random.Random(case["mix"] + 1)
    ways = []
    for m in q_len:
        c = r.randint(1, min(case["kept"], m))
        first = r.randint(1, c)
        if m - c < c - first:
            first = c
        ways.append(list(range(first)) + sorted(r.sample(range(c, m), c - first)))
    return ways


def _params(case):
    """Each row's temperature, top-k (0: all), top-p (1: all) and min-p (0: all): by the case alone."""
    n, r = case["rows"], random.Random(case["mix"])
    if case["params"] == "none":
        return [1.0] * n, [0] * n, [1.0] * n, [0.0] * n
    if case["params"] == "default":
        return [0.7] * n, [40] * n, [0.9] * n, [0.0] * n
    if case["params"] == "top_p":
        return [r.choice([0.6, 0.8, 1.0]) for _ in range(n)], [0] * n, [r.choice([0.8, 0.9, 0.95, 0.99]) for _ in range(n)], [0.0] * n
    # requests of many users: greedy ones, plain ones, each filter by itself and several together
    kinds = [(0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (0.8, 50, 1.0, 0.0), (1.0, 0, 0.95, 0.0), (0.6, 20, 0.95, 0.0), (1.0, 0, 1.0, 0.05), (1.2, 1000, 0.9, 0.02)]
    rows = [r.choice(kinds) for _ in range(n)]
    return tuple(list(x) for x in zip(*rows))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    s = dict(case)
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        s["logits"] = (randn(n, v) * case["spread"]).to(TYPES[case["act"]])
        t, k, p, m = _params(case)
        s["temperature"], s["top_p"], s["min_p"] = (torch.tensor(x, dtype=torch.float32, device="cuda") for x in (t, p, m))
        s["top_k"] = ints(k)
        s["u"] = rand(n)
        s["tokens"] = torch.empty(n, dtype=torch.int32, device="cuda")
        if case["probs"]:
            s["p"] = torch.empty(n, v, device="cuda")
        return s
    q_len, kv_len = _lengths(case)
    n = case["seqs"]
    starts = [0]
    for x in q_len:
        starts.append(starts[-1] + x)
    s["q_start"] = ints(starts)
    s["tokens_n"], s["max_q"], s["max_kv"] = starts[-1], max(q_len), max(kv_len)
    t = starts[-1]
    if case["op"] == "accept":
        parent, _, mask, s["words"] = _trees(case, q_len, seed)
        s["parent"], s["mask"] = ints(parent), mask.cuda()
        s["kv_len"], s["table"] = s["q_start"][1:] - s["q_start"][:-1], torch.zeros(n, 1, dtype=torch.int32, device="cuda")
        s["draft"] = torch.randint(case["vocab"], (t,), generator=g, device="cuda").int()
        # the target's tokens: often the last child's, else any
        s["sampled"] = torch.randint(case["vocab"], (t,), generator=g, device="cuda").int()
        up = s["parent"].long() + torch.repeat_interleave(s["q_start"][:-1].long(), s["kv_len"].long())
        child = torch.where((rand(t) < 0.7) & (s["parent"] >= 0), torch.arange(t, device="cuda"), -1)
        child = torch.full((t,), -1, device="cuda").scatter_reduce_(0, up.clamp(min=0), child, "amax")
        s["sampled"] = torch.where(child >= 0, s["draft"][child.clamp(min=0)], s["sampled"])
        s["path"] = torch.empty(n, s["max_q"], dtype=torch.int32, device="cuda")
        s["tokens"] = torch.empty(n, s["max_q"], dtype=torch.int32, device="cuda")
        s["count"] = torch.empty(n, dtype=torch.int32, device="cuda")
        return s
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    cache = TYPES[case["cache"]]
    need = [-(-x // page) for x in kv_len]
    pages = sum(need) + 3  # a pool with a little room
    width = max(need) + 1
    table = torch.full((n, width), -1, dtype=torch.int32)
    order = torch.randperm(pages, generator=g, device="cuda").int().cpu()
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c]
        at += c
    s["table"], s["kv_len"], s["pages"] = table.cuda(), ints(kv_len), pages
    # [page][head][token][dim] or [page][token][head][dim], of every layer
    shape = (case.get("layers", 1), pages) + ((hk, page, d) if case["by_head"] else (page, hk, d))
    s["k"], s["v"] = randn(*shape).to(cache), randn(*shape).to(cache)
    if case["op"] == "keep":
        way = _ways(case, q_len)
        s["path"], s["count"] = ints([w + [-1] * (case["kept"] - len(w)) for w in way]), ints([len(w) for w in way])
        return s
    h, act = case["heads"], TYPES[case["act"]]
    _, depth, mask, s["words"] = _trees(case, q_len, seed)
    s["depth"], s["mask"] = ints(depth), mask.cuda()
    s["out"] = torch.empty(t, h, d, dtype=act, device="cuda")
    if case["op"] == "append":
        s["qkv"] = randn(t, (h + 2 * hk) * d).to(act)  # the projection's output: queries, keys and values of a token in one row
        if case["norms"]:
            s["q_norm"], s["k_norm"] = 1 + 0.2 * randn(d), 1 + 0.2 * randn(d)
    else:
        s["q"] = randn(t, h, d).to(act)
    return s


# ---- the operators in plain operations ------------------------------------------------


def _rows(s):
    """Each new token's sequence, its sequence's context (tokens before the new ones), its place among the new ones."""
    row = torch.arange(s["tokens_n"], device="cuda")
    start = s["q_start"].long()
    seq = torch.searchsorted(start[1:], row, right=True)
    return seq, (s["kv_len"].long() - (start[1:] - start[:-1]))[seq], row - start[seq]


def _bits(s):
    """Whether a new token sees the i-th new one of its sequence."""
    i = torch.arange(s["max_q"], device="cuda")
    return (s["mask"][:, i // 32] >> (i % 32)) & 1 == 1


def _rotate(x, angle, rot, halves):
    c, sn = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if halves:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat([a * c - b * sn, a * sn + b * c, x[..., rot:]], -1)
    a, b = x[..., :rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2), x[..., rot:]], -1)


def _plain_append(s):
    h, hk, d, rot, page = s["heads"], s["kv_heads"], s["dim"], s["rot"], s["page"]
    t = s["tokens_n"]
    seq, context, i = _rows(s)
    q, k, v = (x.reshape(t, -1, d) for x in s["qkv"].split([h * d, hk * d, hk * d], -1))
    q, k = q.float(), k.float()
    if s["norms"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-5) * s["q_norm"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-5) * s["k_norm"]
    # far positions: the angles need 64 bits
    turn = s["theta"] ** (-2.0 * torch.arange(rot // 2, device="cuda", dtype=torch.float64) / rot)
    angle = (context + s["depth"].long()).double()[:, None] * turn
    s["out"].copy_(_rotate(q, angle, rot, s["halves"]))
    k = _rotate(k, angle, rot, s["halves"]).to(s["k"].dtype)
    at, slot = s["table"][seq, (context + i) // page].long(), (context + i) % page
    if s["by_head"]:
        s["k"][0][at, :, slot] = k
        s["v"][0][at, :, slot] = v.to(s["v"].dtype)
    else:
        s["k"][0][at, slot] = k
        s["v"][0][at, slot] = v.to(s["v"].dtype)
    return s["out"], s["k"], s["v"]


def _plain_attend(s):
    h, hk, d, page, n = s["heads"], s["kv_heads"], s["dim"], s["page"], s["seqs"]
    rep, mq, mk = h // hk, s["max_q"], s["max_kv"]
    seq, _, place = _rows(s)
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    context = kv_len - (start[1:] - start[:-1])
    # every sequence's queries and keys, padded to the longest
    i = torch.arange(mq, device="cuda")
    at = (start[:-1, None] + i).clamp(max=s["tokens_n"] - 1)
    q = s["q"][at].float()
    q = q.reshape(n, mq, hk, rep, d).permute(0, 2, 3, 1, 4).reshape(n, hk, rep * mq, d)
    table = s["table"][:, :-(-mk // page)].long().clamp(min=0)
    j = torch.arange(mk, device="cuda")
    there = (j < kv_len[:, None])[:, None, :, None]

    def taken(pool):
        x = pool[0][table].float()
        x = x.permute(0, 2, 1, 3, 4) if s["by_head"] else x.permute(0, 3, 1, 2, 4)
        return x.reshape(n, hk, -1, d)[:, :, :mk].masked_fill(~there, 0.0)

    score = q @ taken(s["k"]).transpose(-1, -2)
    score *= 1.0 / math.sqrt(d)
    new = j - context[:, None]  # a key's place among the new ones
    bits = _bits(s)[at]
    seen = torch.where((new < 0)[:, None], True, bits.gather(-1, new.clamp(0, mq - 1)[:, None].expand(n, mq, mk)) & (j < kv_len[:, None])[:, None])
    if s["window"]:
        # of the context, what lies less than a window before the token's place in the sequence that its branch makes
        seen = seen & ((new >= 0)[:, None] | (j > (context[:, None] + s["depth"][at])[..., None] - s["window"]))
    score = score.view(n, hk, rep, mq, mk).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score -= torch.where(top == -math.inf, 0.0, top)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    o = score.view(n, hk, rep * mq, mk) @ taken(s["v"])
    o = torch.where(total > 0, o.view(n, hk, rep, mq, d) / total, 0.0).reshape(n, h, mq, d)
    s["out"].copy_(o[seq, :, place])
    return s["out"]


def _plain_sample(s):
    # 64 bits throughout: a draw lies next to a border now and then
    n, v = s["rows"], s["vocab"]
    l = s["logits"].double()
    top = l.amax(-1, keepdim=True)
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    e = torch.where(greedy, (l == top).double(), ((l - top) / torch.where(greedy, 1.0, t)).exp())
    order = l.sort(dim=-1, descending=True, stable=True)[1]  # ties: the lowest index first
    w = e.gather(-1, order)
    rank = torch.arange(v, device="cuda")
    k = s["top_k"].long()[:, None]
    kept = ((rank < k) | (k <= 0)) & (~greedy | (rank < 1))
    w = w * kept
    upto = w.cumsum(-1)
    p = s["top_p"].double()[:, None]
    kept &= (upto - w < p * upto[:, -1:]) | (p >= 1) | (rank < 1)
    kept &= w >= s["min_p"].double()[:, None].clamp(max=1.0)
    left = torch.zeros_like(e).scatter_(-1, order, w * kept)
    cdf = left.cumsum(-1)
    pick = torch.searchsorted(cdf, s["u"].double()[:, None] * cdf[:, -1:], right=True)[:, 0]
    last = v - 1 - (left > 0).flip(-1).int().argmax(-1)
    s["tokens"].copy_(torch.minimum(pick, last))
    if not s["probs"]:
        return s["tokens"]
    s["p"].copy_(left / cdf[:, -1:])
    return s["tokens"], s["p"]


def _plain_accept(s):
    n, mq = s["seqs"], s["max_q"]
    start = s["q_start"].long()
    seq, _, place = _rows(s)
    up = (start[seq] + s["parent"].long()).clamp(min=0)
    follows = (s["parent"] >= 0) & (s["draft"] == s["sampled"][up])
    # of the children that hold the token, the first
    first = torch.full((s["tokens_n"],), mq, device="cuda").scatter_reduce_(0, up, torch.where(follows, place, mq), "amin")
    chosen = (s["parent"] < 0) | (follows & (first[up] == place))
    # a node is on the way if it and all its ancestors are chosen
    chosen = torch.zeros(n, mq, dtype=torch.bool, device="cuda").index_put_((seq, place), chosen)
    on = (chosen[seq] | ~_bits(s)).all(-1)
    way = torch.zeros(n, mq, dtype=torch.bool, device="cuda").index_put_((seq, place), on)
    count = way.sum(-1)
    i = torch.arange(mq, device="cuda")
    path = torch.where(way, i, mq).sort(-1)[0]
    token = s["sampled"][(start[:-1, None] + path).clamp(max=s["tokens_n"] - 1)]
    s["path"].copy_(torch.where(path < mq, path, -1))
    s["tokens"].copy_(torch.where(path < mq, token, -1))
    s["count"].copy_(count)
    return s["path"], s["tokens"], s["count"]


def _plain_keep(s):
    n, page = s["seqs"], s["page"]
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    context = (kv_len - (start[1:] - start[:-1]))[:, None]
    i = torch.arange(s["kept"], device="cuda")
    seq, i = torch.nonzero(i < s["count"][:, None], as_tuple=True)
    to = context[seq, 0] + i
    of = context[seq, 0] + s["path"][seq, i]
    a, b, c, d = s["table"][seq, of // page].long(), of % page, s["table"][seq, to // page].long(), to % page
    if s["by_head"]:
        s["k"][:, c, :, d] = s["k"][:, a, :, b]
        s["v"][:, c, :, d] = s["v"][:, a, :, b]
    else:
        s["k"][:, c, d] = s["k"][:, a, b]
        s["v"][:, c, d] = s["v"][:, a, b]
    return s["k"], s["v"]


# ---- the library's calls --------------------------------------------------------------


def _library():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wasm-chord_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import wcb
    return wcb


def _handles(s, wcb):
    """What a serving program makes once for its cache and once for each step's batch."""
    if "batch" in s:
        return
    kinds = {"f32": wcb.KV_F32, "f16": wcb.KV_F16, "bf16": wcb.KV_BF16}
    s["batch"] = wcb.PagedBatch(s["q_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), s["seqs"], s["tokens_n"], s["max_q"],
                                s["table"].shape[1])
    if "k" in s:
        hk, d, page = s["kv_heads"], s["dim"], s["page"]
        strides = (hk * page * d, d, page * d) if s["by_head"] else (page * hk * d, hk * d, d)
        layers = [wcb.PagedKV(k.data_ptr(), v.data_ptr(), kinds[s["cache"]], s["pages"], page, hk, d, *strides) for k, v in zip(s["k"], s["v"])]
        s["kv"], s["layers_kv"] = layers[0], wcb.PagedLayers(layers)
    if "depth" in s:
        s["tree"] = wcb.PagedTree(s["depth"].data_ptr(), s["mask"].data_ptr(), s["words"])
        s["kind"] = kinds[s["act"]]
    if s["op"] == "append":
        s["rope"] = wcb.Rope(s["rot"], theta=s["theta"], halves=s["halves"])
    elif s["op"] == "attend":
        size = wcb.paged_attention_workspace(s["kv"], s["batch"], s["heads"])
        s["room"] = torch.zeros(size, dtype=torch.uint8, device="cuda")


def _own_append(s, wcb):
    _handles(s, wcb)
    h, hk, d, qkv = s["heads"], s["kv_heads"], s["dim"], s["qkv"]
    at, size, row = qkv.data_ptr(), qkv.element_size(), (h + 2 * hk) * d
    norms = (s["q_norm"].data_ptr(), s["k_norm"].data_ptr()) if s["norms"] else (0, 0)
    wcb.paged_tree_append_dev(s["kv"], s["batch"], s["tree"], s["rope"], at, at + h * d * size, at + (h + hk) * d * size, s["out"].data_ptr(), s["kind"], h,
                              row, row, row, h * d, *norms, 1e-5, torch.cuda.current_stream().cuda_stream)
    return s["out"], s["k"], s["v"]


def _own_attend(s, wcb):
    _handles(s, wcb)
    row = s["heads"] * s["dim"]
    wcb.paged_tree_attention_dev(s["kv"], s["batch"], s["tree"], s["q"].data_ptr(), s["out"].data_ptr(), s["kind"], s["heads"], row, row, s["room"].data_ptr(),
                                 s["room"].numel(), window=s["window"], stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_sample(s, wcb):
    if "set" not in s:
        s["set"] = wcb.Sampling(s["temperature"].data_ptr(), s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr())
        s["kind"] = {"f32": wcb.KV_F32, "f16": wcb.KV_F16, "bf16": wcb.KV_BF16}[s["act"]]
    wcb.sample_dev(s["logits"].data_ptr(), s["kind"], s["rows"], s["vocab"], s["set"], s["u"].data_ptr(), s["tokens"].data_ptr(),
                   probs_ptr=s["p"].data_ptr() if s["probs"] else 0, stream=torch.cuda.current_stream().cuda_stream)
    return (s["tokens"], s["p"]) if s["probs"] else s["tokens"]


def _own_accept(s, wcb):
    _handles(s, wcb)
    wcb.tree_accept_dev(s["batch"], s["parent"].data_ptr(), s["draft"].data_ptr(), s["sampled"].data_ptr(), s["max_q"], s["path"].data_ptr(),
                        s["tokens"].data_ptr(), s["count"].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    return s["path"], s["tokens"], s["count"]


def _own_keep(s, wcb):
    _handles(s, wcb)
    wcb.paged_keep_dev(s["layers_kv"], s["batch"], s["path"].data_ptr(), s["kept"], s["count"].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    return s["k"], s["v"]


def run(state):
    if own:
        return {"append": _own_append, "attend": _own_attend, "sample": _own_sample, "accept": _own_accept, "keep": _own_keep}[state["op"]](state, _library())
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample, "accept": _plain_accept, "keep": _plain_keep}[state["op"]](state)


def work(case):
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        return {"bytes": float(n * (v * ((4 if case["act"] == "f32" else 2) + (4 if case["probs"] else 0)) + 24)), "flops": float(4 * n * v)}
    q_len, kv_len = _lengths(case)
    t = sum(q_len)
    if case["op"] == "accept":  # parents, drafted and sampled tokens; the way, its tokens, its length
        return {"bytes": float(12 * t + case["seqs"] * (8 * max(q_len) + 8)), "flops": float(t)}
    hk, d = case["kv_heads"], case["dim"]
    c = 4 if case["cache"] == "f32" else 2
    if case["op"] == "keep":  # the tokens that move: read once, written once, in all layers
        moved = sum(i != j for w in _ways(case, q_len) for i, j in enumerate(w))
        return {"bytes": float(case["layers"] * moved * 2 * 2 * hk * d * c + 4 * case["seqs"] * (case["kept"] + 1)), "flops": 0.0}
    h = case["heads"]
    a = 4 if case["act"] == "f32" else 2
    table = 4 * sum(-(-x // case["page"]) for x in kv_len)
    words = -(-max(q_len) // 32)
    if case["op"] == "append":
        return {"bytes": float(t * (2 * h * d * a + 2 * hk * d * (a + c) + 4) + 8 * case["seqs"]), "flops": float(t * d * (h + hk) * (7 if case["norms"] else 3))}
    seen = keys = 0
    for q, kv in zip(q_len, kv_len):
        w = min(case["window"] or kv, kv - q)
        seen += q * w + q * min(q, 6)  # the context, and a branch of the tree
        keys += w + q
    return {"bytes": float(2 * t * h * d * a + 2 * keys * hk * d * c + table + 4 * t * (words + 1)), "flops": 4.0 * h * d * seen}


# ---- the operators in 64 bits, each sequence by itself --------------------------------


def exact(case, seed):
    f64 = torch.float64
    if case["op"] == "accept":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "keep":
        q_len, kv_len = _lengths(case)
        table, page = s["table"].tolist(), case["page"]
        pools = []
        for pool in (s["k"], s["v"]):
            x = (pool.transpose(2, 3) if case["by_head"] else pool).to(f64)  # [layer][page][slot][head][dim]
            for i, way in enumerate(_ways(case, q_len)):
                at = [(table[i][(kv_len[i] - q_len[i] + j) // page], (kv_len[i] - q_len[i] + j) % page) for j in way + list(range(len(way)))]
                a, b = (torch.tensor(y, device="cuda") for y in zip(*at))
                m = len(way)
                x[:, a[m:], b[m:]] = x[:, a[:m], b[:m]].clone()
            pools.append(x.transpose(2, 3) if case["by_head"] else x)
        return pools[0], pools[1]
    if case["op"] == "sample":
        if not case["probs"]:
            return None
        p = torch.zeros(case["rows"], case["vocab"], dtype=f64, device="cuda")
        for i, (t, k, top_p, min_p) in enumerate(zip(*_params(case))):
            x = s["logits"][i].to(f64)
            if t <= 0:
                p[i, int((x == x.max()).nonzero()[0])] = 1.0
                continue
            # by the probabilities themselves: the largest ones, ties in the order of their indices
            q = torch.softmax(x / torch.tensor(t, dtype=torch.float32).to(f64).item(), -1)
            order = torch.argsort(-x, stable=True)
            order = order[:k] if k > 0 else order
            r = q[order] / q[order].sum()
            if top_p < 1:
                at = torch.searchsorted(r.cumsum(0), torch.tensor(top_p, dtype=torch.float32, device="cuda").to(f64))
                order = order[:int(at) + 1]
            order = order[q[order] >= torch.tensor(min_p, dtype=torch.float32).to(f64).item() * q.max()]
            p[i, order] = q[order] / q[order].sum()
        return None, p
    q_len, kv_len = _lengths(case)
    h, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    table = s["table"].cpu()
    depth, words = s["depth"].cpu(), s["mask"].cpu().long()

    def slots(i, first, last):
        """Where tokens first .. last - 1 of sequence i lie, as places of a pool with its tokens in one axis."""
        p = torch.arange(first, last)
        return (table[i, p // page].long() * page + p % page).cuda()

    def by_token(pool):
        x = pool[0].transpose(1, 2) if case["by_head"] else pool[0]
        return x.reshape(-1, hk, d)

    if case["op"] == "attend":
        k, v = by_token(s["k"]), by_token(s["v"])
        out = torch.zeros(s["tokens_n"], h, d, dtype=f64, device="cuda")
        r0 = 0
        for i, (nq, nk) in enumerate(zip(q_len, kv_len)):
            at, context = slots(i, 0, nk), nk - nq
            seen = torch.ones(nq, nk, dtype=torch.bool)
            for r in range(nq):
                seen[r, context:] = torch.tensor([int(words[r0 + r, j // 32]) >> (j % 32) & 1 for j in range(nq)]).bool()
                if case["window"]:
                    seen[r, :min(context, max(0, context + int(depth[r0 + r]) - case["window"] + 1))] = False
            seen = seen.cuda()
            for head in range(h):
                kk, vv = (x[at, head * hk // h].to(f64) for x in (k, v))
                a = s["q"][r0:r0 + nq, head].to(f64) @ kk.T / d ** 0.5
                out[r0:r0 + nq, head] = torch.softmax(a.masked_fill_(~seen, -math.inf), -1) @ vv
            r0 += nq
        return out
    rot = case["rot"]
    k, v = by_token(s["k"]).to(f64), by_token(s["v"]).to(f64)
    x = s["qkv"].to(f64).view(s["tokens_n"], h + 2 * hk, d)
    turn = [case["theta"] ** (-2 * m / rot) for m in range(rot // 2)]
    first = torch.arange(rot // 2) if case["halves"] else 2 * torch.arange(rot // 2)
    second = first + rot // 2 if case["halves"] else first + 1
    made = []
    r0 = 0
    for i, (nq, nk) in enumerate(zip(q_len, kv_len)):
        part = x[r0:r0 + nq].clone()
        if case["norms"]:
            for lo, hi, w in ((0, h, s["q_norm"]), (h, h + hk, s["k_norm"])):
                y = part[:, lo:hi]
                part[:, lo:hi] = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.to(f64)
        where = (nk - nq + depth[r0:r0 + nq]).to(f64).cuda()
        a = where[:, None, None] * torch.tensor(turn, dtype=f64, device="cuda")
        z = torch.polar(torch.ones_like(a), a) * torch.complex(part[:, :h + hk, first], part[:, :h + hk, second])
        part[:, :h + hk, first], part[:, :h + hk, second] = z.real, z.imag
        at = slots(i, nk - nq, nk)
        k[at], v[at] = part[:, h:h + hk], part[:, h + hk:]
        made.append(part[:, :h])
        r0 += nq
    back = (lambda y: y.view(1, s["pages"], page, hk, d).transpose(2, 3)) if case["by_head"] else (lambda y: y.view(1, s["pages"], page, hk, d))
    return torch.cat(made), back(k), back(v)
