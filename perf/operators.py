"""Cases of the paged serving operators, for measurement and comparison.

Three operators carry a serving step over a paged key/value cache:

- append: the new tokens' queries and keys are normalised for each head (where the
  model has such norms) and rotated by their positions; keys and values go to their
  pages, queries to an output;
- attend: the new tokens (one, a few drafted ones, or a prompt's chunk) attend to
  their sequence's pages, causally, optionally within a window;
- verify: drafted tokens are accepted or replaced by the target's probabilities, from
  given random numbers.

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
        # one new token of a short chat: the call's latency (TinyLlama heads, the f16 cache under f32 activations)
        {"name": "append one token", "op": "append", "seqs": 1, "q_min": 1, "q_max": 1, "kv_min": 333, "kv_max": 333, "heads": 32,
         "kv_heads": 4, "dim": 64, "rot": 64, "halves": False, "norms": False, "theta": 10000.0, "act": "f32", "cache": "f16", "page": 16, "by_head": True, "mix": 1},
        # a batch of drafted tokens far into their sequences, norms of queries and keys, 70B heads
        {"name": "append drafts", "op": "append", "seqs": 32, "q_min": 1, "q_max": 6, "kv_min": 40, "kv_max": 4096, "heads": 64,
         "kv_heads": 8, "dim": 128, "rot": 128, "halves": True, "norms": True, "theta": 500000.0, "act": "bf16", "cache": "bf16", "page": 16, "by_head": False, "mix": 2},
        # prompts' chunks, 7B heads
        {"name": "append prompts", "op": "append", "seqs": 7, "q_min": 301, "q_max": 1500, "kv_min": 301, "kv_max": 1500, "heads": 32,
         "kv_heads": 32, "dim": 128, "rot": 128, "halves": False, "norms": False, "theta": 10000.0, "act": "f16", "cache": "f16", "page": 64, "by_head": False, "mix": 3},
        # one token of one short sequence: latency
        {"name": "attend one token", "op": "attend", "seqs": 1, "q_min": 1, "q_max": 1, "kv_min": 333, "kv_max": 333, "heads": 32,
         "kv_heads": 4, "dim": 64, "act": "f32", "cache": "f16", "page": 16, "by_head": True, "window": 0, "mix": 4},
        # a full serving batch, one token each, ragged lengths, 70B heads
        {"name": "attend decode batch", "op": "attend", "seqs": 64, "q_min": 1, "q_max": 1, "kv_min": 1, "kv_max": 8191, "heads": 64,
         "kv_heads": 8, "dim": 128, "act": "bf16", "cache": "bf16", "page": 16, "by_head": False, "window": 0, "mix": 5},
        # one token at the end of a very long document
        {"name": "attend long decode", "op": "attend", "seqs": 1, "q_min": 1, "q_max": 1, "kv_min": 131071, "kv_max": 131071, "heads": 64,
         "kv_heads": 8, "dim": 128, "act": "f16", "cache": "f16", "page": 64, "by_head": True, "window": 0, "mix": 6},
        # drafted tokens to be verified, 7B heads (no sharing of keys)
        {"name": "attend drafts", "op": "attend", "seqs": 16, "q_min": 1, "q_max": 6, "kv_min": 500, "kv_max": 2304, "heads": 32,
         "kv_heads": 32, "dim": 128, "act": "f16", "cache": "f16", "page": 32, "by_head": False, "window": 0, "mix": 7},
        # a prompt's chunk at the end of a long context, 70B heads
        {"name": "attend prompt chunk", "op": "attend", "seqs": 1, "q_min": 2047, "q_max": 2047, "kv_min": 32767, "kv_max": 32767, "heads": 64,
         "kv_heads": 8, "dim": 128, "act": "bf16", "cache": "bf16", "page": 64, "by_head": False, "window": 0, "mix": 8},
        # prompts and single tokens in one batch, a sliding window, the f32 cache of the reference's numerics, TinyLlama heads
        {"name": "attend mixed f32", "op": "attend", "seqs": 9, "q_min": 1, "q_max": 700, "kv_min": 1, "kv_max": 1500, "heads": 32,
         "kv_heads": 4, "dim": 64, "act": "f32", "cache": "f32", "page": 16, "by_head": True, "window": 511, "mix": 9},
        # one user's drafts: latency
        {"name": "verify one", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 32000, "sampled": True, "mix": 10},
        # a serving batch whose drafts come without probabilities (a lookup's tokens)
        {"name": "verify lookup batch", "op": "verify", "seqs": 32, "drafts": 7, "vocab": 32000, "sampled": False, "mix": 11},
        # a large batch over a large vocabulary of odd size
        {"name": "verify large batch", "op": "verify", "seqs": 192, "drafts": 5, "vocab": 100003, "sampled": True, "mix": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "verify"])
    mix = rng.randrange(1 << 30)
    if op == "verify":
        vocab = _spread(rng, 1000, 131072)
        drafts = rng.randint(1, 8)
        seqs = _spread(rng, 1, max(1, min(192, 100_000_000 // (vocab * (drafts + 1)))))
        return {"op": op, "seqs": seqs, "drafts": drafts, "vocab": vocab, "sampled": rng.random() < 0.7, "mix": mix}
    heads, kv_heads, dim = rng.choice([(32, 4, 64), (32, 32, 128), (64, 8, 128), (8, 2, 64), (15, 5, 64), (8, 1, 128)])
    act, cache = rng.choice([("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "bf16")])
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "act": act, "cache": cache, "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 128]),
            "by_head": rng.random() < 0.5, "mix": mix}
    if op == "append":
        case["seqs"] = _spread(rng, 1, 48)
        case["q_max"] = _spread(rng, 1, max(1, min(2048, 4000 // case["seqs"])))
        case["kv_max"] = case["q_max"] + _spread(rng, 1, 2000)
        case["kv_min"] = case["q_max"]
        case.update(rot=dim if rng.random() < 0.7 else dim // 2, halves=rng.random() < 0.5, norms=rng.random() < 0.5, theta=rng.choice([10000.0, 500000.0]))
    else:
        case["seqs"] = _spread(rng, 1, 64)
        kind = rng.choice(["one", "few", "many"])
        case["q_max"] = 1 if kind == "one" else rng.randint(2, 17) if kind == "few" else _spread(rng, 18, 1024)
        # the plain form holds seqs x longest chunk x longest sequence x heads scores, and its sequences' keys in 32 bits
        most = min(600_000_000 // (case["seqs"] * case["q_max"] * heads), 130_000_000 // (case["seqs"] * kv_heads * dim), 60000)
        case["kv_max"] = max(case["q_max"], _spread(rng, 1, max(2, most)))
        case["kv_min"] = max(1, case["kv_max"] // 8)
        case["window"] = 0 if rng.random() < 0.7 else _spread(rng, 1, max(2, case["kv_max"]))
    case["q_min"] = 1 if rng.random() < 0.7 else case["q_max"]
    return case


def _lengths(case):
    """New tokens and cached tokens (new ones included) of each sequence: by the case alone."""
    r = random.Random(case["mix"])
    q = [r.randint(case["q_min"], case["q_max"]) for _ in range(case["seqs"])]
    kv = [max(n, r.randint(case["kv_min"], case["kv_max"])) for n in q]
    q[0] = case["q_max"]
    kv[0] = max(q[0], case["kv_max"])
    return q, kv


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    s = dict(case)
    if case["op"] == "verify":
        n, k, v = case["seqs"], case["drafts"], case["vocab"]
        logits = randn(n, k + 1, v) * 2.5
        s["target"] = torch.softmax(logits, -1)
        if case["sampled"]:  # the draft model is near the target's
            s["draft_probs"] = torch.softmax(logits[:, :k].add_(randn(n, k, v) * 0.7), -1)
            pick = s["draft_probs"]
        else:  # a lookup that is right now and then
            pick = s["target"][:, :k]
        cdf = pick.double().cumsum(-1)
        at = torch.searchsorted(cdf, rand(n, k, 1).double() * cdf[..., -1:], right=True).clamp_(max=v - 1)
        s["draft"] = at[..., 0].int().contiguous()
        if not case["sampled"]:
            top = s["target"][:, :k].argmax(-1).int()
            s["draft"] = torch.where(rand(n, k) < 0.8, top, s["draft"]).contiguous()
        r = random.Random(case["mix"])
        lens = [r.randint(max(1, k // 2), k) for _ in range(n)]
        s["draft_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["u_accept"], s["u_sample"] = rand(n, k), rand(n)
        s["tokens"] = torch.empty(n, k + 1, dtype=torch.int32, device="cuda")
        s["accepted"] = torch.empty(n, dtype=torch.int32, device="cuda")
        return s
    q_len, kv_len = _lengths(case)
    n, h, hk, d, page = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    act, cache = TYPES[case["act"]], TYPES[case["cache"]]
    need = [-(-x // page) for x in kv_len]
    pages = sum(need) + 3  # a pool with a little room
    width = max(need) + 1
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((n, width), -1, dtype=torch.int32)
    order = order.cpu()
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c]
        at += c
    s["table"] = table.cuda()
    starts = [0]
    for x in q_len:
        starts.append(starts[-1] + x)
    s["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    s["tokens_n"], s["max_q"], s["max_kv"], s["pages"] = starts[-1], max(q_len), max(kv_len), pages
    t = starts[-1]
    # [page][head][token][dim] or [page][token][head][dim]
    shape = (pages, hk, page, d) if case["by_head"] else (pages, page, hk, d)
    s["k"], s["v"] = randn(*shape).to(cache), randn(*shape).to(cache)
    s["q_out"] = torch.empty(t, h, d, dtype=act, device="cuda")
    if case["op"] == "append":
        s["qkv"] = randn(t, (h + 2 * hk) * d).to(act)  # the projection's output: queries, keys and values of a token in one row
        if case["norms"]:
            s["q_norm"], s["k_norm"] = 1 + 0.2 * randn(d), 1 + 0.2 * randn(d)
    else:
        s["q"] = randn(t, h, d).to(act)
        s["out"] = s["q_out"]
    return s


# ---- the operators in plain operations ------------------------------------------------


def _rows(s):
    """Each new token's sequence and position."""
    row = torch.arange(s["tokens_n"], device="cuda")
    seq = torch.searchsorted(s["q_start"][1:].long(), row, right=True)
    q_len = (s["q_start"][1:] - s["q_start"][:-1]).long()
    return row, seq, s["kv_len"].long()[seq] - q_len[seq] + row - s["q_start"].long()[seq]


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
    _, seq, pos = _rows(s)
    q, k, v = (x.reshape(t, -1, d) for x in s["qkv"].split([h * d, hk * d, hk * d], -1))
    q, k = q.float(), k.float()
    if s["norms"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-5) * s["q_norm"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-5) * s["k_norm"]
    # far positions: the angles need 64 bits
    angle = pos.double()[:, None] * s["theta"] ** (-2.0 * torch.arange(rot // 2, device="cuda", dtype=torch.float64) / rot)
    s["q_out"].copy_(_rotate(q, angle, rot, s["halves"]))
    k = _rotate(k, angle, rot, s["halves"]).to(s["k"].dtype)
    at, slot = s["table"][seq, pos // page].long(), pos % page
    if s["by_head"]:
        s["k"][at, :, slot] = k
        s["v"][at, :, slot] = v.to(s["v"].dtype)
    else:
        s["k"][at, slot] = k
        s["v"][at, slot] = v.to(s["v"].dtype)
    return s["q_out"], s["k"], s["v"]


def _plain_attend(s):
    h, hk, d, page, n = s["heads"], s["kv_heads"], s["dim"], s["page"], s["seqs"]
    rep, mq, mk = h // hk, s["max_q"], s["max_kv"]
    row, seq, _ = _rows(s)
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    q_len = start[1:] - start[:-1]
    # every sequence's queries and keys, padded to the longest
    i = torch.arange(mq, device="cuda")
    q = s["q"][(start[:-1, None] + i).clamp(max=s["tokens_n"] - 1)].float()
    q = q.reshape(n, mq, hk, rep, d).permute(0, 2, 3, 1, 4).reshape(n, hk, rep * mq, d)
    table = s["table"][:, :-(-mk // page)].long().clamp(min=0)
    j = torch.arange(mk, device="cuda")
    there = (j < kv_len[:, None])[:, None, :, None]

    def taken(pool):
        x = pool[table].float()
        x = x.permute(0, 2, 1, 3, 4) if s["by_head"] else x.permute(0, 3, 1, 2, 4)
        return x.reshape(n, hk, -1, d)[:, :, :mk].masked_fill(~there, 0.0)

    score = q @ taken(s["k"]).transpose(-1, -2)
    score *= 1.0 / math.sqrt(d)
    pos = (kv_len - q_len)[:, None] + i
    seen = (j <= pos[..., None]) & (j < kv_len[:, None, None])
    if s["window"]:
        seen &= j > pos[..., None] - s["window"]
    score = score.view(n, hk, rep, mq, mk).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score -= torch.where(top == -math.inf, 0.0, top)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    o = score.view(n, hk, rep * mq, mk) @ taken(s["v"])
    o = torch.where(total > 0, o.view(n, hk, rep, mq, d) / total, 0.0).reshape(n, h, mq, d)
    s["out"].copy_(o[seq, :, row - start[seq]])
    return s["out"]


def _plain_verify(s):
    n, k, v = s["seqs"], s["drafts"], s["vocab"]
    each, i = torch.arange(n, device="cuda"), torch.arange(k, device="cuda")
    at = s["draft"].long()[..., None]
    p = s["target"][:, :k].gather(-1, at)[..., 0].double()
    q = s["draft_probs"].gather(-1, at)[..., 0].double() if s["sampled"] else torch.ones_like(p)
    length = s["draft_len"].long()
    fine = (s["u_accept"].double() * q < p) & (i < length[:, None])
    count = fine.long().cumprod(-1).sum(-1)
    left = s["target"][each, count].double()
    short = count < length
    if s["sampled"]:
        less = s["draft_probs"][each, count.clamp(max=k - 1)].double()
    else:
        less = torch.nn.functional.one_hot(s["draft"].long()[each, count.clamp(max=k - 1)], v).double()
    rest = torch.where(short[:, None], (left - less).clamp_(min=0.0), left)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, left)
    cdf = rest.cumsum(-1)
    pick = torch.searchsorted(cdf, s["u_sample"].double()[:, None] * cdf[:, -1:], right=True)[:, 0]
    last = (v - 1 - (rest > 0).flip(-1).int().argmax(-1))
    pick = torch.minimum(pick, last)
    j = torch.arange(k + 1, device="cuda")
    drafted = torch.nn.functional.pad(s["draft"].long(), (0, 1))
    tokens = torch.where(j < count[:, None], drafted, torch.where(j == count[:, None], pick[:, None], -1))
    s["tokens"].copy_(tokens)
    s["accepted"].copy_(count)
    return s["tokens"], s["accepted"]


# ---- the library's calls --------------------------------------------------------------


def _library():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wasm-chord_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import wcb
    return wcb


def _handles(s, wcb):
    """What a serving program makes once for its cache and once for each step's batch."""
    if "kv" not in s:
        kinds = {"f32": wcb.KV_F32, "f16": wcb.KV_F16, "bf16": wcb.KV_BF16}
        hk, d, page = s["kv_heads"], s["dim"], s["page"]
        strides = (hk * page * d, d, page * d) if s["by_head"] else (page * hk * d, hk * d, d)
        s["kv"] = wcb.PagedKV(s["k"].data_ptr(), s["v"].data_ptr(), kinds[s["cache"]], s["pages"], page, hk, d, *strides)
        s["batch"] = wcb.PagedBatch(s["q_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), s["seqs"], s["tokens_n"], s["max_q"],
                                    s["table"].shape[1])
        s["kind"] = kinds[s["act"]]
        if s["op"] == "append":
            s["rope"] = wcb.Rope(s["rot"], theta=s["theta"], halves=s["halves"])
        else:
            size = wcb.paged_attention_workspace(s["kv"], s["batch"], s["heads"])
            s["room"] = torch.zeros(size, dtype=torch.uint8, device="cuda")


def _own_append(s, wcb):
    _handles(s, wcb)
    h, hk, d, qkv = s["heads"], s["kv_heads"], s["dim"], s["qkv"]
    at, size, row = qkv.data_ptr(), qkv.element_size(), (h + 2 * hk) * d
    norms = (s["q_norm"].data_ptr(), s["k_norm"].data_ptr()) if s["norms"] else (0, 0)
    wcb.paged_append_dev(s["kv"], s["batch"], s["rope"], at, at + h * d * size, at + (h + hk) * d * size, s["q_out"].data_ptr(), s["kind"], h,
                         row, row, row, h * d, *norms, 1e-5, torch.cuda.current_stream().cuda_stream)
    return s["q_out"], s["k"], s["v"]


def _own_attend(s, wcb):
    _handles(s, wcb)
    row = s["heads"] * s["dim"]
    wcb.paged_attention_dev(s["kv"], s["batch"], s["q"].data_ptr(), s["out"].data_ptr(), s["kind"], s["heads"], row, row, s["room"].data_ptr(),
                            s["room"].numel(), window=s["window"], stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_verify(s, wcb):
    wcb.spec_verify_dev(s["draft"].data_ptr(), s["draft_len"].data_ptr(), s["target"].data_ptr(), s["draft_probs"].data_ptr() if s["sampled"] else 0,
                        s["u_accept"].data_ptr(), s["u_sample"].data_ptr(), s["seqs"], s["drafts"], s["vocab"], s["tokens"].data_ptr(),
                        s["accepted"].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    return s["tokens"], s["accepted"]


def run(state):
    if own:
        return {"append": _own_append, "attend": _own_attend, "verify": _own_verify}[state["op"]](state, _library())
    return {"append": _plain_append, "attend": _plain_attend, "verify": _plain_verify}[state["op"]](state)


def work(case):
    if case["op"] == "verify":
        # one row of probabilities of each sequence is searched, less its draft's where a token was turned down, and the drafted tokens' own are looked at
        n, k, v = case["seqs"], case["drafts"], case["vocab"]
        rows = 2 if case["sampled"] else 1
        return {"bytes": float(n * (4 * v * rows + 4 * (5 * k + 5))), "flops": float(n * v * (rows + 1))}
    q_len, kv_len = _lengths(case)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    a, c, t = (4 if case["act"] == "f32" else 2), (4 if case["cache"] == "f32" else 2), sum(q_len)
    table = 4 * sum(-(-x // case["page"]) for x in kv_len)
    if case["op"] == "append":
        return {"bytes": float(t * (2 * h * d * a + 2 * hk * d * (a + c)) + 8 * case["seqs"]), "flops": float(t * d * (h + hk) * (7 if case["norms"] else 3))}
    seen = keys = 0
    for q, kv in zip(q_len, kv_len):
        w = case["window"] or kv
        seen += sum(min(p + 1, w) for p in range(kv - q, kv))
        keys += min(kv, w + q - 1)
    return {"bytes": float(2 * t * h * d * a + 2 * keys * hk * d * c + table), "flops": 4.0 * h * d * seen}


# ---- the operators in 64 bits, each sequence by itself --------------------------------


def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers
    s = prepare(case, seed)
    q_len, kv_len = _lengths(case)
    h, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    table = s["table"].cpu()
    f64 = torch.float64

    def slots(i, first, last):
        """Where tokens first .. last - 1 of sequence i lie, as places of a pool with its tokens in one axis."""
        p = torch.arange(first, last)
        return (table[i, p // page].long() * page + p % page).cuda()

    def by_token(pool):
        x = pool.transpose(1, 2) if case["by_head"] else pool
        return x.reshape(-1, hk, d)

    if case["op"] == "attend":
        k, v = by_token(s["k"]), by_token(s["v"])
        out = torch.zeros(s["tokens_n"], h, d, dtype=f64, device="cuda")
        r0 = 0
        for i, (nq, nk) in enumerate(zip(q_len, kv_len)):
            at = slots(i, 0, nk)
            ahead = torch.arange(nk, device="cuda")[None, :] - torch.arange(nk - nq, nk, device="cuda")[:, None]
            hidden = ahead > 0
            if case["window"]:
                hidden = hidden | (ahead <= -case["window"])
            for head in range(h):
                kk, vv = (x[at, head * hk // h].to(f64) for x in (k, v))
                a = s["q"][r0:r0 + nq, head].to(f64) @ kk.T / d ** 0.5
                out[r0:r0 + nq, head] = torch.softmax(a.masked_fill_(hidden, -math.inf), -1) @ vv
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
        a = torch.arange(nk - nq, nk, dtype=f64, device="cuda")[:, None, None] * torch.tensor(turn, dtype=f64, device="cuda")
        z = torch.polar(torch.ones_like(a), a) * torch.complex(part[:, :h + hk, first], part[:, :h + hk, second])
        part[:, :h + hk, first], part[:, :h + hk, second] = z.real, z.imag
        at = slots(i, nk - nq, nk)
        k[at], v[at] = part[:, h:h + hk], part[:, h + hk:]
        made.append(part[:, :h])
        r0 += nq
    back = (lambda y: y.view(s["pages"], page, hk, d).transpose(1, 2)) if case["by_head"] else (lambda y: y.view(s["pages"], page, hk, d))
    return torch.cat(made), back(k), back(v)
