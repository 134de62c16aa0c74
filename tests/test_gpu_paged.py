"""Paged serving operators on the GPU against plain 64-bit forms: append
(wcb_paged_append_dev), attention (wcb_paged_attention_dev), verification of
drafted tokens (wcb_spec_verify_dev), and the three of them as one step."""
import math

import numpy as np
import pytest

import wcb

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

KIND = {"f32": (torch.float32, wcb.KV_F32), "f16": (torch.float16, wcb.KV_F16), "bf16": (torch.bfloat16, wcb.KV_BF16)}
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


def half_step(t):
    return torch.finfo(t).eps / 2


class _Slots:
    """Where a sequence's tokens lie in a [pages][page] pool."""

    def __init__(self, row, page, n):
        t = np.arange(n)
        self.a, self.b = torch.from_numpy(row[t // page].astype(np.int64)), torch.from_numpy(t % page)

    def __len__(self):
        return len(self.a)


class _View:
    """A pool as [pages][page][heads][dim], read and written by _Slots."""

    def __init__(self, t):
        self.t = t

    def __getitem__(self, s):
        return self.t[s.a, s.b]

    def __setitem__(self, s, v):
        if len(s):
            self.t[s.a, s.b] = v


class Step:
    """A pool, its sequences and the new tokens' rows. Everything of no sequence holds `junk`."""

    def __init__(self, q_len, kv_len, heads=8, kv_heads=2, dim=64, act="f32", cache="f16", page=16, by_head=False, seed=0, junk=float("nan"), extra=3,
                 first=0, gap=0, width=None):
        g = torch.Generator().manual_seed(seed)
        self.q_len, self.kv_len, self.h, self.hk, self.d, self.page = list(q_len), list(kv_len), heads, kv_heads, dim, page
        self.act, self.cache = act, cache
        self.at, self.ak = KIND[act]
        self.ct, self.ck = KIND[cache]
        n = len(q_len)
        need = [-(-max(x, 0) // page) for x in kv_len]
        self.pages = sum(need) + 2
        order = torch.randperm(self.pages, generator=g).tolist()
        width = width or max(need + [1]) + 1
        table = np.full((n, width), -7, np.int32)
        p = 0
        for i, c in enumerate(need):
            table[i, :c] = order[p:p + c]
            p += c
        self.table = table
        start = [first]
        for x in q_len:
            start.append(start[-1] + x)
        self.start = start
        self.tokens = start[-1] + extra  # rows behind the last sequence
        shape = (self.pages, kv_heads, page, dim) if by_head else (self.pages, page, kv_heads, dim)
        self.by_head = by_head
        k, v = torch.full(shape, junk), torch.full(shape, junk)
        kt, vt = self.by_token(k), self.by_token(v)
        for i in range(n):
            s = self.slots(i)
            kt[s] = torch.randn(len(s), kv_heads, dim, generator=g)
            vt[s] = torch.randn(len(s), kv_heads, dim, generator=g)
        self.k, self.v = k.to(self.ct).cuda(), v.to(self.ct).cuda()
        # rows with a gap between tokens
        self.row = heads * dim + gap
        self.q = torch.randn(self.tokens, self.row, generator=g).to(self.at).cuda()
        self.out = torch.full((self.tokens, self.row), 7.0, dtype=self.at, device="cuda")
        self.lse = torch.full((self.tokens, heads), 7.0, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.upload()

    def upload(self):
        self.dev = [torch.tensor(np.asarray(x), dtype=torch.int32).cuda() for x in (self.start, self.kv_len, self.table)]
        self.kv = self.describe()
        self.batch = wcb.PagedBatch(*[x.data_ptr() for x in self.dev], len(self.q_len), self.tokens, max(max(self.q_len), 1), self.table.shape[1],
                                    self.status.data_ptr())

    def describe(self):
        s = (self.hk * self.page * self.d, self.d, self.page * self.d) if self.by_head else (0, 0, 0)
        return wcb.PagedKV(self.k.data_ptr(), self.v.data_ptr(), self.ck, self.pages, self.page, self.hk, self.d, *s)

    def by_token(self, pool):
        return _View(pool.transpose(1, 2) if self.by_head else pool)

    def slots(self, i):
        return _Slots(self.table[i], self.page, max(0, self.kv_len[i]))

    def workspace(self):
        n = wcb.paged_attention_workspace(self.kv, self.batch, self.h)
        w = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
        w[:4096] = 0
        return w

    def attend(self, window=0, scale=0.0, room=None, stream=0, lse=True):
        room = self.workspace() if room is None else room
        wcb.paged_attention_dev(self.kv, self.batch, self.q.data_ptr(), self.out.data_ptr(), self.ak, self.h, self.row, self.row, room.data_ptr(),
                                room.numel(), scale=scale, window=window, lse_ptr=self.lse.data_ptr() if lse else 0, stream=stream)
        return room

    def expected(self, window=0, scale=0.0):
        """out, lse and each output's tolerance, in 64 bits."""
        scale = scale or 1 / math.sqrt(self.d)
        rep = self.h // self.hk
        q = self.q[:, :self.h * self.d].double().cpu().view(-1, self.h, self.d)
        kt, vt = self.by_token(self.k.cpu().double()), self.by_token(self.v.cpu().double())
        out = torch.full(q.shape, 7.0, dtype=torch.float64)
        lse = torch.full(q.shape[:2], 7.0, dtype=torch.float64)
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        e = half_step(self.at)
        for i, (nq, nk) in enumerate(zip(self.q_len, self.kv_len)):
            s = self.slots(i)
            k, v = kt[s].repeat_interleave(rep, 1), vt[s].repeat_interleave(rep, 1)
            pos = torch.arange(nk - nq, nk)[:, None]
            j = torch.arange(max(nk, 0))[None]
            seen = (j <= pos) & ((j > pos - window) if window else True)
            rows = q[self.start[i]:self.start[i] + nq]
            if nk <= 0:
                out[self.start[i]:self.start[i] + nq], lse[self.start[i]:self.start[i] + nq] = 0, -math.inf
            if nq == 0 or nk <= 0:
                continue
            a = torch.einsum("qhd,khd->hqk", rows, k.nan_to_num()) * scale
            # each product of 64 or 128 terms in 32 bits, terms split to 21 bits for f32 activations (2^-21 with both splits)
            da = torch.einsum("qhd,khd->hqk", rows.abs(), k.nan_to_num().abs()) * abs(scale) * ((self.d + 8) * 2.0 ** -24 + (2.0 ** -20 if self.act == "f32" else 0))
            a = a.masked_fill(~seen, -math.inf)
            l = a.logsumexp(-1) if nk > 0 else torch.full(a.shape[:2], -math.inf, dtype=torch.float64)
            p = torch.where(seen, (a - torch.where(l == -math.inf, 0.0, l)[..., None]).exp(), 0.0)
            # NaN in a place that some row does not see: only the others get it
            vz = v.nan_to_num(0, 0, 0)
            o = torch.einsum("hqk,khd->qhd", p, vz)
            # p: 2 da from its score (and the sum's), 2^-21 from the exponential, one rounding to the 16-bit type where it is
            # rounded once, and 2^-24 of the largest (f16's subnormals)
            dp = p * (4 * da.amax(-1, keepdim=True).nan_to_num() + 2.0 ** -20 + (e if self.act != "f32" else 2.0 ** -21)) + (2.0 ** -24 * p.amax(-1, keepdim=True) if self.act == "f16" else 0) * seen
            t = torch.einsum("hqk,khd->qhd", dp, vz.abs()) + e * o.abs() * 1.01 + 1e-30 + (nk * 2.0 ** -24) * torch.einsum("hqk,khd->qhd", p, vz.abs())
            r = slice(self.start[i], self.start[i] + nq)
            out[r], lse[r] = o, l.T
            tol[r] = t
            ltol[r] = (2 * da.amax(-1) + 2.0 ** -20).T + (l.abs().T.nan_to_num(0, 0, 0) + 8) * 2.0 ** -22
        return out, lse, tol, ltol

    def check(self, window=0, scale=0.0, status=0):
        out, lse, tol, ltol = self.expected(window, scale)
        got = self.out[:, :self.h * self.d].double().cpu().view(out.shape)
        err = (got - out).abs()
        assert torch.isfinite(got).all()
        assert (err <= tol).all(), ((err / tol.clamp(min=1e-300)).max(), err.max())
        gl = self.lse.double().cpu()
        same = (gl == lse) | ((gl - lse).abs() <= ltol)
        assert same.all(), (gl - lse).abs().max()
        assert int(self.status.item()) == status
        if self.row > self.h * self.d:
            assert (self.out[:, self.h * self.d:] == 7.0).all()


# ---- attention ------------------------------------------------------------------------

@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 4, 128), (16, 1, 128), (15, 5, 64)])
@pytest.mark.parametrize("page,by_head", [(16, False), (24, True), (1, False)])
def test_attention_of_single_tokens(gpu, act, cache, heads, kv_heads, dim, page, by_head):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300]
    s = Step([1] * len(lens), lens, heads, kv_heads, dim, act, cache, page, by_head, seed=1)
    s.attend()
    s.check()


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 4, 128), (16, 1, 128), (15, 5, 64), (40, 1, 64)])
@pytest.mark.parametrize("q_len,kv_len", [([2, 5, 1, 0, 3], [40, 5, 70, 9, 130]), ([17, 1, 64, 33], [17, 200, 191, 100]), ([150, 1, 7], [150, 33, 260])])
def test_attention_of_chunks(gpu, act, cache, heads, kv_heads, dim, q_len, kv_len):
    s = Step(q_len, kv_len, heads, kv_heads, dim, act, cache, 16, True, seed=2, gap=16, first=2)
    s.attend()
    s.check()


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("window", [1, 2, 50, 64, 1000])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_window(gpu, act, cache, window, dim):
    s = Step([1, 40, 3, 129], [400, 300, 3, 129], 8, 2, dim, act, cache, 32, False, seed=3)
    s.attend(window=window)
    s.check(window=window)


@pytest.mark.parametrize("act,cache", PAIRS)
def test_rows_that_see_nothing_are_zero(gpu, act, cache):
    # no keys at all; fewer keys than new tokens (the first ones have negative positions)
    s = Step([1, 5, 2], [0, 3, 20], 8, 2, 64, act, cache, 16, seed=4)
    s.attend()
    s.check(status=wcb.PAGED_BAD_LEN)
    assert (s.out[0] == 0).all() and (s.out[1:3] == 0).all() and torch.isinf(s.lse[0:3]).all()


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (8, 8, 128)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_values_of_unseen_keys_do_not_reach_a_row(gpu, act, cache, heads, kv_heads, dim, what):
    # the last new token's key and value, and one out of the window of all but the first
    q, kv, window = [70, 3], [140, 30], 60
    s = Step(q, kv, heads, kv_heads, dim, act, cache, 16, seed=5)
    clean = Step(q, kv, heads, kv_heads, dim, act, cache, 16, seed=5)
    for x in (s.k, s.v):
        for i, j in ((0, 139), (0, 11), (1, 29)):
            x[int(s.table[i, j // 16]), j % 16] = what
    s.attend(window=window)
    clean.attend(window=window)
    assert int(s.status.item()) == 0
    # rows 0..68 of the first sequence do not see key 139; only row 0 (position 70) sees key 11 (11 > 70 - 60)
    for r in [*range(1, 69), 70, 71]:
        assert torch.equal(s.out[r], clean.out[r]), r
    for r in (0, 69, 72):
        if what == what and what < 0:
            continue  # a key of -infinity may have no weight
        assert not torch.isfinite(s.out[r].float()).any()


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f16", "f16")])
def test_bad_pages_take_no_part(gpu, act, cache):
    s = Step([1, 40], [100, 120], 8, 2, 64, act, cache, 16, seed=6)
    want = s.table.copy()
    s.table[0, 2], s.table[1, 0], s.table[1, 7] = -1, s.pages, 1 << 30
    s.upload()
    s.attend()
    assert int(s.status.item()) == wcb.PAGED_BAD_PAGE
    # the same with those keys masked, by 64-bit softmax over the others
    q = s.q.double().cpu().view(-1, 8, 64)
    s.table = want
    kt, vt = s.by_token(s.k.cpu().double()), s.by_token(s.v.cpu().double())
    for i, r, pos, holes in ((0, 0, 99, [2]), (1, 1, 80, [0, 7]), (1, 40, 119, [0, 7])):
        j = torch.arange(s.kv_len[i])
        seen = (j <= pos) & ~torch.isin(j // 16, torch.tensor(holes))
        sl = s.slots(i)
        a = torch.einsum("hd,khd->hk", q[r], kt[sl].repeat_interleave(4, 1)) / 8
        p = a.masked_fill(~seen, -math.inf).softmax(-1)
        o = torch.einsum("hk,khd->hd", p, vt[sl].repeat_interleave(4, 1))
        # values of a few units: 4 roundings of p and o in the type, and the scores' 32 bits
        assert ((s.out[r].double().cpu().view(8, 64) - o).abs() <= 4 * max(half_step(s.at), 2e-6)).all()


def test_lengths_past_the_page_table(gpu):
    s = Step([2, 1], [40, 20], 8, 2, 64, "f16", "f16", 16, seed=7)
    s.table = s.table[:, :2].copy()  # 32 tokens a sequence
    s.upload()
    s.attend()
    assert int(s.status.item()) == wcb.PAGED_BAD_PAGE
    t = Step([2, 1], [40, 20], 8, 2, 64, "f16", "f16", 16, seed=7)
    out, *_ = t.expected()
    assert (s.out[2].double().cpu().view(8, 64) - out[2]).abs().max() <= 2e-3 and torch.isfinite(s.out[:2].float()).all()


@pytest.mark.parametrize("start", [[0, 5, 3, 6], [-1, 2, 4, 6], [0, 2, 4, 99], [0, 1 << 30, 4, 6]])
def test_unsound_rows_are_skipped(gpu, start):
    s = Step([2, 2, 2], [40, 20, 30], 8, 2, 64, "f16", "f16", 16, seed=8, extra=0)
    s.start = start
    s.upload()
    s.attend()
    assert int(s.status.item()) & wcb.PAGED_BAD_ROWS
    for i in range(3):
        lo, hi = start[i], start[i + 1]
        sound = 0 <= lo <= hi <= 6
        if not sound and 0 <= lo < 6 and not any(0 <= a <= lo < b <= 6 for a, b in zip(start, start[1:])):
            assert (s.out[lo] == 7.0).all()


def test_more_sequences_than_threads(gpu):
    n = 700
    q = [(i * 7) % 4 for i in range(n)]
    kv = [max(x, (i * 37) % 90) for i, x in enumerate(q)]
    s = Step(q, kv, 8, 2, 64, "bf16", "bf16", 16, seed=9)
    s.attend()
    s.check()


# units of one, two and many tiles, so many of them that parts begin and end in units of each kind
@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("dim,chunks", [(64, False), (128, False), (64, True), (128, True)])
def test_short_and_long_units(gpu, act, cache, dim, chunks):
    n = 60 if chunks else 300
    q = [(1, 40, 3, 70, 0, 130, 33)[i % 7] if chunks else 1 for i in range(n)]
    kv = [x + (0, 100, 20, 250, 60, 1, 700, 127, 128, 64, 900)[i % 11] for i, x in enumerate(q)]
    s = Step(q, kv, 8, 4, dim, act, cache, 32, False, seed=31)
    s.attend()
    s.check()


# one sequence cut into about 7, 8, 9, 16, 17, 127 .. 130 and 256 pieces: joined in one go, by groups, by large groups
@pytest.mark.parametrize("act,cache,dim", [("f16", "f16", 128), ("f32", "f32", 64), ("f32", "bf16", 64)])
@pytest.mark.parametrize("kv", [448, 512, 513, 1024, 1025, 8128, 8192, 8256, 8257, 16384])
def test_pieces_and_groups(gpu, act, cache, dim, kv):
    s = Step([1], [kv], 8, 2, dim, act, cache, 64, True, seed=32)
    room = s.attend()
    s.check()
    first = s.out.clone()
    s.attend(room=room)
    assert torch.equal(first, s.out) and (room[:4096] == 0).all()


@pytest.mark.parametrize("act,cache,heads,kv_heads,dim", [("f16", "f16", 8, 2, 128), ("f32", "f16", 32, 4, 64), ("bf16", "bf16", 64, 8, 128)])
def test_long_sequences_and_repeatability(gpu, act, cache, heads, kv_heads, dim):
    s = Step([1, 1], [20011, 3], heads, kv_heads, dim, act, cache, 64, True, seed=10)
    room = s.attend()
    s.check()
    first, lse = s.out.clone(), s.lse.clone()
    for _ in range(5):
        s.out.fill_(7.0)
        s.attend(room=room)
        assert torch.equal(first, s.out) and torch.equal(lse, s.lse)  # joined in a fixed order
    assert (room[:4096] == 0).all()


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim,page,by_head", [(8, 1, 128, 64, False), (4, 4, 128, 16, True), (8, 2, 64, 48, False), (15, 5, 64, 1, True)])
@pytest.mark.parametrize("q_len,kv_len,window", [([257], [2600], 0), ([129, 1, 300, 0, 64], [129, 70, 1500, 5, 640], 0), ([200, 333], [900, 333], 130)])
def test_attention_of_long_chunks(gpu, act, cache, heads, kv_heads, dim, page, by_head, q_len, kv_len, window):
    s = Step(q_len, kv_len, heads, kv_heads, dim, act, cache, page, by_head, seed=16, gap=8)
    room = s.attend(window=window)
    s.check(window=window)
    first, lse = s.out.clone(), s.lse.clone()
    for _ in range(3):
        s.out.fill_(7.0)
        s.attend(window=window, room=room)
        assert torch.equal(first, s.out) and torch.equal(lse, s.lse)
    assert (room[:4096] == 0).all()


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("dim", [64, 128])
def test_growing_scores_rescale(gpu, act, cache, dim):
    """Scores that grow along the keys by far more than 2^8: the sums are rescaled again and again."""
    s = Step([140, 1], [900, 700], 4, 2, dim, act, cache, 16, seed=17)
    s.q.abs_()
    for i in range(2):
        sl = s.slots(i)
        ramp = torch.linspace(-4, 4, len(sl))[:, None, None]
        k = s.by_token(s.k.float().cpu())
        k[sl] = k[sl] * 0.1 + ramp
        s.k.copy_(k.t.transpose(1, 2) if s.by_head else k.t)
    s.attend()
    s.check()
    s.attend(scale=-0.3)
    s.check(scale=-0.3)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_len", [1, 90, 300])
@pytest.mark.parametrize("qs,ks,vs", [(1e-20, 1e18, 1e-25), (1e20, 1e-21, 1e30), (1.0, 1.0, 1.0)])
def test_f32_of_any_range(gpu, dim, q_len, qs, ks, vs):
    """f32 queries, keys and values far from 1, and sizes that differ from key to key."""
    s = Step([q_len], [400], 4, 2, dim, "f32", "f32", 16, seed=18)
    g = torch.Generator().manual_seed(5)
    j = torch.exp2(torch.randint(-6, 1, (s.pages, 16, 1, 1), generator=g).float()).cuda()
    s.q *= qs
    s.k *= ks * j
    s.v *= vs * j.flip(0)
    s.attend()
    s.check()


def test_scale_and_large_scores(gpu):
    s = Step([3, 1], [100, 50], 8, 2, 64, "f32", "f32", 16, seed=11)
    s.attend(scale=-3.0)
    s.check(scale=-3.0)


def test_pages_beyond_32_bit_offsets(gpu):
    """A pool whose last page starts past 2^32 elements; K and V share it."""
    page, hk, d = 64, 2, 128
    pages = (1 << 32) // (page * hk * d) + 3
    pool = torch.empty(pages, page, hk, d, dtype=torch.float16, device="cuda")
    small = Step([1], [200], 4, hk, d, "f16", "f16", page, seed=12)
    ids = [pages - 1, 0, pages // 2 + 1, pages - 2]
    for i, p in enumerate(ids):
        pool[p] = small.k[int(small.table[0, i])]
    small.v = small.k
    small.kv = small.describe()
    small.attend()
    want = small.out.clone()
    table = torch.tensor([ids + [-1]], dtype=torch.int32, device="cuda")
    kv = wcb.PagedKV(pool.data_ptr(), pool.data_ptr(), wcb.KV_F16, pages, page, hk, d)
    b = wcb.PagedBatch(small.dev[0].data_ptr(), small.dev[1].data_ptr(), table.data_ptr(), 1, small.tokens, 1, 5)
    room = small.workspace()
    small.out.fill_(7.0)
    wcb.paged_attention_dev(kv, b, small.q.data_ptr(), small.out.data_ptr(), wcb.KV_F16, 4, small.row, small.row, room.data_ptr(), room.numel())
    assert torch.equal(small.out, want)


def test_attention_in_a_graph_follows_the_lengths(gpu):
    s = Step([1, 1, 6], [300, 41, 90], 8, 2, 64, "f16", "f16", 16, seed=13, width=40)
    room = s.attend()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.attend(room=room, stream=torch.cuda.current_stream().cuda_stream)
    for kv in ([300, 40, 90], [17, 41, 89], [299, 3, 6]):
        s.dev[1].copy_(torch.tensor(kv, dtype=torch.int32))
        s.kv_len = kv
        s.out.fill_(7.0)
        s.lse.fill_(7.0)
        graph.replay()
        s.check()


FIRST_CALL = """
import sys
sys.path.insert(0, {pkg!r}); sys.path.insert(0, {tests!r})
import torch, wcb
import test_gpu_paged as t
for act, cache in t.PAIRS:
    for q_len in ([1, 2], [90, 3]):
        s = t.Step(q_len, [300, 40], 8, 2, 64, act, cache, 16, seed=40)
        room, side, graph = s.workspace(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.attend(room=room, stream=torch.cuda.current_stream().cuda_stream)
        graph.replay()
        graph.replay()
        s.check()
print("captured first")
"""


def test_the_first_call_may_be_a_captured_one(gpu):
    """Every kernel's set-up on its first call is allowed while a stream is captured: in a process of its own."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = FIRST_CALL.format(pkg=os.path.join(os.path.dirname(here), "wasm-chord_b200"), tests=here)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


def test_two_graphs_share_a_workspace(gpu):
    """Replayed one after the other, in either order: a call leaves its workspace as it found it."""
    a = Step([1, 30], [3000, 500], 8, 2, 128, "f16", "f16", 16, seed=41)
    b = Step([4, 1, 200], [900, 2500, 800], 8, 2, 128, "f16", "f16", 16, seed=42)
    room = max((a.workspace(), b.workspace()), key=lambda w: w.numel())
    graphs = []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.attend(room=room, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for order in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for s in (a, b):
            s.out.fill_(7.0)
            s.lse.fill_(7.0)
        for i in order:
            graphs[i].replay()
        a.check()
        b.check()


@pytest.mark.parametrize("act", ["f32", "f16"])
def test_largest_and_smallest_batches(gpu, act):
    """Sequences without new tokens only; a padded batch; the longest row counts wrong on the host's side."""
    s = Step([0, 0, 0], [5, 0, 100], 8, 2, 64, act, "f16", 16, seed=43)
    s.attend()
    assert (s.out == 7.0).all() and (s.lse == 7.0).all()
    s = Step([3, 70, 1], [40, 90, 7], 8, 2, 64, act, "f16", 16, seed=44, extra=50)
    s.batch._c.max_q_len = 1  # the largest is 70
    s.attend()
    s.check()


def test_two_streams_with_a_workspace_each(gpu):
    a = Step([1, 30], [3000, 500], 8, 2, 128, "f16", "f16", 16, seed=14)
    b = Step([4, 1], [900, 2500], 8, 2, 128, "f16", "f16", 16, seed=15)
    ra, rb = a.workspace(), b.workspace()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        a.attend(room=ra, stream=sa.cuda_stream)
        b.attend(room=rb, stream=sb.cuda_stream)
    torch.cuda.synchronize()
    a.check()
    b.check()


# ---- append ---------------------------------------------------------------------------

def rotated(x, pos, rot, halves, inv_freq):
    """x [tokens][heads][dim] in 64 bits."""
    x = x.clone()
    a = pos.double()[:, None] * torch.tensor(inv_freq, dtype=torch.float64)
    c, sn = a.cos()[:, None], a.sin()[:, None]
    i = torch.arange(rot // 2)
    f, g = (i, i + rot // 2) if halves else (2 * i, 2 * i + 1)
    p, q = x[..., f].clone(), x[..., g].clone()
    x[..., f], x[..., g] = p * c - q * sn, p * sn + q * c
    return x


def check_append(s, rot, halves, norms, theta=10000.0, inv_freq=None, in_place=False, fused=True, status=0, eps=1e-5, n_heads=None):
    g = torch.Generator().manual_seed(99)
    h, hk, d, t = s.h, s.hk, s.d, s.tokens
    width = (h + 2 * hk) * d + 16
    qkv = torch.randn(t, width, generator=g).to(s.at).cuda()
    before = qkv.clone()
    wq, wk = (1 + 0.3 * torch.randn(d, generator=g)).cuda(), (1 + 0.3 * torch.randn(d, generator=g)).cuda()
    q_out = qkv if in_place else torch.full((t, h * d + 32), 7.0, dtype=s.at, device="cuda")
    k0, v0 = s.k.clone(), s.v.clone()
    es = qkv.element_size()
    rope = wcb.Rope(rot, theta=theta, halves=halves, inv_freq=inv_freq) if rot else None
    p = qkv.data_ptr()
    wcb.paged_append_dev(s.kv, s.batch, rope, p, p + h * d * es, p + (h + hk) * d * es, q_out.data_ptr(), s.ak, h, width, width, width,
                         width if in_place else h * d + 32, wq.data_ptr() if norms else 0, wk.data_ptr() if norms else 0, eps)
    torch.cuda.synchronize()
    inv = list(rope._c.inv_freq[:rot // 2]) if rot else []
    x = before[:, :(h + 2 * hk) * d].double().cpu().view(t, h + 2 * hk, d)
    wantk, wantv = s.by_token(k0.double().cpu()), s.by_token(v0.double().cpu())
    keep_q = before if in_place else torch.full_like(q_out, 7.0)
    want_q = keep_q[:, :h * d].double().cpu().view(t, h, d)
    tolk = torch.zeros_like(wantk.t)
    written = torch.zeros(t, dtype=torch.bool)
    for i, (nq, nk) in enumerate(zip(s.q_len, s.kv_len)):
        r = slice(s.start[i], s.start[i] + nq)
        written[r] = True
        pos = torch.arange(nk - nq, nk)
        q, k, v = x[r, :h].clone(), x[r, h:h + hk].clone(), x[r, h + hk:]
        if norms:
            q = q / (q.square().mean(-1, keepdim=True) + eps).sqrt() * wq.double().cpu()
            k = k / (k.square().mean(-1, keepdim=True) + eps).sqrt() * wk.double().cpu()
        if rot:
            q, k = rotated(q, pos, rot, halves, inv), rotated(k, pos, rot, halves, inv)
        want_q[r] = q
        for j, pp in enumerate(pos.tolist()):
            if 0 <= pp < s.table.shape[1] * s.page and 0 <= s.table[i, pp // s.page] < s.pages:
                a, b = int(s.table[i, pp // s.page]), pp % s.page
                wantk.t[a, b], wantv.t[a, b] = k[j], v[j]
                tolk[a, b] = 1
    # f32 arithmetic on values of a few units (the sum of 128 squares, two products, sine and cosine of a turn: 2^-20
    # together), then one rounding
    ref = x.abs().amax() * 4
    got = q_out[:, :h * d].double().cpu().view(t, h, d)
    assert ((got - want_q).abs() <= half_step(s.at) * want_q.abs() * 1.01 + written[:, None, None] * 2.0 ** -20 * ref).all()
    if not in_place:
        assert (q_out[:, h * d:] == 7.0).all()
    else:
        assert torch.equal(qkv[:, h * d:], before[:, h * d:])
    gk, gv = s.by_token(s.k.double().cpu()).t, s.by_token(s.v.double().cpu()).t
    same = lambda a, b: torch.equal(a.nan_to_num(123.0), b.nan_to_num(123.0))
    assert same(gk[tolk == 0], wantk.t[tolk == 0]) and same(gv[tolk == 0], wantv.t[tolk == 0])  # nothing else is written
    w = tolk == 1
    assert ((gk[w] - wantk.t[w]).abs() <= half_step(s.ct) * wantk.t[w].abs() * 1.01 + 2.0 ** -20 * ref).all()
    assert torch.equal(gv[w].to(s.ct), wantv.t[w].to(s.ct))  # values are only rounded
    assert int(s.status.item()) == status


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 4, 128), (15, 5, 64)])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("rot,norms,page,by_head", [(1, False, 16, True), (1, True, 24, False), (0.5, True, 1, False), (0.25, False, 16, False), (0, True, 16, True)])
def test_append(gpu, act, cache, heads, kv_heads, dim, halves, rot, norms, page, by_head):
    rot = int(dim * rot)
    s = Step([1, 5, 0, 33], [1, 40, 9, 100], heads, kv_heads, dim, act, cache, page, by_head, seed=20, first=1)
    check_append(s, rot - rot % 16, halves, norms)


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("halves", [False, True])
def test_append_in_place(gpu, act, cache, halves):
    check_append(Step([1, 5, 400], [1, 40, 400], 8, 2, 128, act, cache, 16, seed=21), 128, halves, True, in_place=True)


def test_append_far_positions(gpu):
    # angles of 10^6 radians and more: 32 bits would be off by 0.06
    s = Step([3, 1], [1000003, 99], 8, 2, 64, "f32", "f32", 4096, seed=22)
    check_append(s, 64, False, False, theta=1e6)


def test_append_given_frequencies_and_many_sequences(gpu):
    n = 600
    s = Step([(i * 5) % 3 for i in range(n)], [2 + (i * 11) % 60 for i in range(n)], 8, 2, 64, "f16", "f16", 16, seed=23)
    check_append(s, 32, True, False, inv_freq=[0.3 / (i + 1) for i in range(16)])


def test_append_skips_what_has_no_place(gpu):
    s = Step([3, 2, 2], [2, 40, 30], 8, 2, 64, "f16", "f16", 16, seed=24)  # the first token of sequence 0 has position -1
    s.table[1, 2], s.table[2, 1] = -1, s.pages
    s.upload()
    check_append(s, 64, False, False, status=wcb.PAGED_BAD_LEN | wcb.PAGED_BAD_PAGE)


def test_append_keys_and_values_only(gpu):
    s = Step([2], [20], 8, 2, 64, "f16", "f16", 16, seed=25)
    kv = torch.randn(s.tokens, 2, 2, 64).half().cuda()
    wcb.paged_append_dev(s.kv, s.batch, None, 0, kv.data_ptr(), kv.data_ptr() + 256, 0, wcb.KV_F16, 0, 0, 256, 256, 0)
    sl = s.slots(0)
    assert torch.equal(s.by_token(s.k.cpu())[sl][18:], kv[:2, 0].cpu()) and torch.equal(s.by_token(s.v.cpu())[sl][18:], kv[:2, 1].cpu())


# ---- verification ---------------------------------------------------------------------

def verify_plain(draft, lens, target, probs, ua, us):
    """The definition, one sequence after another, in 64 bits."""
    n, k = draft.shape
    v = target.shape[-1]
    clean = lambda x: np.where((x > 0) & np.isfinite(x), x, 0).astype(np.float64)
    tokens, acc = np.full((n, k + 1), -1, np.int64), np.zeros(n, np.int64)
    for s in range(n):
        m = k if lens is None else min(max(int(lens[s]), 0), k)
        c = 0
        while c < m:
            x = int(draft[s, c])
            if not 0 <= x < v:
                break
            p = clean(target[s, c, x])
            q = clean(probs[s, c, x]) if probs is not None else 1.0
            if not float(ua[s, c]) * float(q) < float(p):
                break
            tokens[s, c] = x
            c += 1
        acc[s] = c
        r = clean(target[s, c])
        if c < m:
            if probs is not None:
                w = np.maximum(r - clean(probs[s, c]), 0)
            else:
                w = r.copy()
                if 0 <= draft[s, c] < v:
                    w[draft[s, c]] = max(0.0, w[draft[s, c]] - 1.0)
            if w.sum() > 0:
                r = w
        if not r.sum() > 0:
            continue
        u = min(max(float(us[s]), 0.0), float(np.float32(1 - 2.0 ** -24))) if us[s] == us[s] else 0.0
        cdf = np.cumsum(r)
        hit = np.nonzero(cdf > u * cdf[-1])[0]
        tokens[s, c] = hit[0] if len(hit) else np.nonzero(r)[0][-1]
    return tokens, acc


def run_verify(draft, lens, target, probs, ua, us, pad=0, status=None):
    n, k = draft.shape
    v = target.shape[-1]
    dev = lambda a, t: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(t).cuda()
    d, l, a, u = dev(draft, torch.int32), dev(lens, torch.int32), dev(ua, torch.float32), dev(us, torch.float32)
    wide = lambda x: None if x is None else torch.nn.functional.pad(torch.from_numpy(x).float().cuda(), (0, pad)).contiguous()
    t, p = wide(target), wide(probs)
    tokens = torch.full((n + 1, k + 1), 77, dtype=torch.int32, device="cuda")
    acc = torch.full((n + 1,), 77, dtype=torch.int32, device="cuda")
    ptr = lambda x: 0 if x is None else x.data_ptr()
    wcb.spec_verify_dev(ptr(d), ptr(l), ptr(t), ptr(p), ptr(a), ptr(u), n, k, v, tokens.data_ptr(), acc.data_ptr(), target_row_stride=v + pad,
                        draft_row_stride=v + pad, status_ptr=ptr(status))
    assert (tokens[n] == 77).all() and acc[n] == 77
    return tokens[:n].cpu().numpy(), acc[:n].cpu().numpy()


def probs_of(rng, *shape, sharp=2.5):
    x = np.exp(sharp * rng.standard_normal(shape))
    return (x / x.sum(-1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("n,k,v", [(1, 1, 1), (1, 4, 32000), (3, 2, 255), (5, 7, 257), (2, 40, 300), (33, 5, 1000), (400, 3, 97), (2, 3, 131072), (6, 0, 500), (17, 4, 50001)])
@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("pad", [0, 3])
def test_verify(gpu, n, k, v, sampled, pad):
    rng = np.random.default_rng(n * 1000 + k)
    target = probs_of(rng, n, k + 1, v)
    probs = (target[:, :k] * np.exp(0.5 * rng.standard_normal((n, k, v)))).astype(np.float32) if k else None
    if k:
        probs /= probs.sum(-1, keepdims=True)
    base = probs if k else target[:, :0]
    draft = np.array([[rng.choice(v, p=(r := row.astype(np.float64)) / r.sum()) for row in m] for m in base], np.int64).reshape(n, k)
    lens = None if n % 2 else rng.integers(0, k + 1, n)
    ua, us = rng.random((n, k), np.float32), rng.random(n, np.float32)
    if not sampled:
        draft = np.where(rng.random((n, k)) < 0.7, target[:, :k].argmax(-1), draft)
        ua *= 0.3
        probs = None
    want = verify_plain(draft, lens, target, probs, ua, us)
    got = run_verify(draft, lens, target, probs, ua, us, pad)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])


def test_verify_edges(gpu):
    v = 5000
    rng = np.random.default_rng(5)
    target, probs = probs_of(rng, 10, 3, v), probs_of(rng, 10, 2, v)
    draft = rng.integers(0, v, (10, 2))
    ua, us = rng.random((10, 2), np.float32), rng.random(10, np.float32)
    draft[0, 0], draft[1, 1], draft[2, 0] = -1, v, 1 << 30       # no tokens of the vocabulary
    ua[1, 0], us[1] = 0.0, 1.0                                    # u = 0 accepts all that is possible; u = 1 is held below 1
    ua[3], us[3] = np.nan, np.nan                                 # comparisons with NaN are false
    target[4] = 0                                                 # nothing to draw from
    probs[5] = target[5, :2]                                      # all accepted
    ua[6], probs[6], target[6, 0] = 1.0, target[6, :2] * 2, 0     # nothing left of the target, and nothing in it
    ua[7], probs[7] = 1.0, target[7, :2] * 2                      # nothing left: from the target itself
    target[8, :, ::3], probs[8, :, ::7] = np.nan, np.inf          # count as zero
    target[9] = 0
    target[9, :, 4999] = 1                                        # a greedy target, the last token
    us[9] = 0.0
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = verify_plain(draft, None, target, probs, ua, us)
    got = run_verify(draft, None, target, probs, ua, us, status=status)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])
    assert int(status.item()) == wcb.PAGED_BAD_TOKEN | wcb.PAGED_BAD_PROBS
    assert got[0][4].tolist() == [-1, -1, -1] and got[0][9, got[1][9]] == 4999


def test_verified_tokens_follow_the_target(gpu):
    """Drafts from q, verified: the first token's distribution is p, not q (20000 sequences, 8 tokens; a
    count's standard deviation is at most sqrt(20000 / 4) = 71: five of them)."""
    n, v = 20000, 8
    rng = np.random.default_rng(6)
    p, q = probs_of(rng, v, sharp=1.0), probs_of(rng, v, sharp=1.0)
    draft = rng.choice(v, size=(n, 1), p=q.astype(np.float64) / q.astype(np.float64).sum())
    target, probs = np.broadcast_to(p, (n, 2, v)).copy(), np.broadcast_to(q, (n, 1, v)).copy()
    tokens, _ = run_verify(draft, None, target, probs, rng.random((n, 1), np.float32), rng.random(n, np.float32))
    count = np.bincount(tokens[:, 0], minlength=v)
    assert np.abs(count - n * p).max() <= 5 * math.sqrt(n / 4)


# ---- a step of a serving loop ---------------------------------------------------------

@pytest.mark.parametrize("cache", ["f32", "f16"])
def test_a_speculative_step(gpu, cache):
    """Append, attend, verify for a ragged batch, captured as one graph and replayed with the next step's inputs; the attention agrees
    with the library's attention over contiguous caches (wcb_attention_dev), whose numbers come from another kernel."""
    h, hk, d, v, k = 32, 4, 64, 2000, 3
    q_len = [k + 1] * 3
    s = Step(q_len, [80, 40, 360], h, hk, d, "f32", cache, 16, True, seed=30, extra=0)  # pages for the tokens to come
    s.kv_len = [54, 11, 337]
    s.upload()
    g = torch.Generator(device="cuda").manual_seed(31)
    t, width = s.tokens, (h + 2 * hk) * d
    qkv = torch.randn(t, width, generator=g, device="cuda")
    q = torch.empty(t, h * d, device="cuda")
    wout = torch.randn(h * d, v, generator=g, device="cuda") * 0.05
    probs = torch.softmax(torch.randn(3, k, v, generator=g, device="cuda"), -1)
    draft = torch.randint(0, v, (3, k), generator=g, device="cuda", dtype=torch.int32)
    ua, us = torch.rand(3, k, generator=g, device="cuda"), torch.rand(3, generator=g, device="cuda")
    tokens, acc = torch.empty(3, k + 1, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    target = torch.empty(3, k + 1, v, device="cuda")
    rope, room = wcb.Rope(d), s.workspace()

    def step():
        st = torch.cuda.current_stream().cuda_stream
        p = qkv.data_ptr()
        wcb.paged_append_dev(s.kv, s.batch, rope, p, p + 4 * h * d, p + 4 * (h + hk) * d, q.data_ptr(), wcb.KV_F32, h, width, width, width, h * d, stream=st)
        wcb.paged_attention_dev(s.kv, s.batch, q.data_ptr(), s.out.data_ptr(), wcb.KV_F32, h, h * d, s.row, room.data_ptr(), room.numel(), stream=st)
        target.copy_(torch.softmax((s.out @ wout).view(3, k + 1, v), -1))
        wcb.spec_verify_dev(draft.data_ptr(), 0, target.data_ptr(), probs.data_ptr(), ua.data_ptr(), us.data_ptr(), 3, k, v, tokens.data_ptr(), acc.data_ptr(), stream=st)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(3):
        qkv.copy_(torch.randn(t, width, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = verify_plain(draft.cpu().numpy(), None, target.cpu().numpy(), probs.cpu().numpy(), ua.cpu().numpy(), us.cpu().numpy())
        assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(acc.cpu().numpy(), want[1])
        for i in range(3):
            n, m = q_len[i], s.kv_len[i]
            sl = s.slots(i)
            kc = torch.zeros(hk, 512, d)
            vc = torch.zeros(hk, 512, d)
            kc[:, :m] = s.by_token(s.k.cpu())[sl].float().transpose(0, 1)
            vc[:, :m] = s.by_token(s.v.cpu())[sl].float().transpose(0, 1)
            kc, vc = kc.cuda(), vc.cuda()
            o = torch.empty(n, h * d, device="cuda")
            rows = q[s.start[i]:s.start[i] + n].contiguous()
            wcb.attention_dev(rows.data_ptr(), kc.data_ptr(), vc.data_ptr(), o.data_ptr(), n, h, hk, d, 512, m, m - n)
            assert (o - s.out[s.start[i]:s.start[i] + n]).abs().max() <= 2e-5 * o.abs().max()
        # the next step: what was accepted and the drawn token stay, the other drafts are overwritten
        s.kv_len = [m - k + int(a) + k + 1 for m, a in zip(s.kv_len, acc)]
        s.dev[1].copy_(torch.tensor(s.kv_len, dtype=torch.int32))
