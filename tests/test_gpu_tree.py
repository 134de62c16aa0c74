"""Trees of drafted tokens on the GPU against plain 64-bit forms: append by depth (wcb_paged_tree_append_dev), attention by
mask (wcb_paged_tree_attention_dev), acceptance (wcb_tree_accept_dev), keeping the accepted tokens (wcb_paged_keep_dev), and
all of them with sampling as the steps of a serving loop."""
import math

import numpy as np
import pytest

import wcb
from test_gpu_paged import PAIRS, Step, half_step, rotated
from test_gpu_sample import sample_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def random_tree(rng, n, near=8):
    return [-1] + [int(rng.randint(max(0, i - near), i)) for i in range(1, n)]


class Tree(Step):
    """A Step whose new tokens are trees: parent lists, or rows of any mask (`masks`: [n][n] truth values of each sequence)."""

    def __init__(self, q_len, kv_len, *a, masks=None, words=None, near=8, **o):
        super().__init__(q_len, kv_len, *a, **o)
        rng = np.random.RandomState(o.get("seed", 0))
        self.parent = [random_tree(rng, n, near) if n else [] for n in q_len]
        self.words = words or max(1, -(-max(q_len) // 32))
        self.sees, self.depths = [], []
        depth = np.full(self.tokens, 1 << 30, np.int32)  # rows of no sequence hold anything
        mask = np.full((self.tokens, self.words), 0xffffffff, np.uint32)
        for i, n in enumerate(q_len):
            see, d = np.zeros((n, n), bool), np.zeros(n, int)
            for j in range(n):
                if self.parent[i][j] >= 0:
                    see[j], d[j] = see[self.parent[i][j]], d[self.parent[i][j]] + 1
                see[j, j] = True
            if masks is not None:
                see = np.asarray(masks[i], bool)
            see[:, 32 * self.words:] = False
            r = slice(self.start[i], self.start[i] + n)
            depth[r] = d
            for w in range(self.words):
                bits = see[:, 32 * w:32 * w + 32].astype(np.uint64)
                mask[r, w] = (bits << np.arange(bits.shape[1], dtype=np.uint64)).sum(-1).astype(np.uint32)
            self.sees.append(torch.from_numpy(see))
            self.depths.append(torch.from_numpy(d))
        self.tree_dev = [torch.from_numpy(depth).cuda(), torch.from_numpy(mask.view(np.int32)).cuda()]
        self.tree = wcb.PagedTree(self.tree_dev[0].data_ptr(), self.tree_dev[1].data_ptr(), self.words)

    def attend(self, window=0, scale=0.0, room=None, stream=0, lse=True):
        room = self.workspace() if room is None else room
        wcb.paged_tree_attention_dev(self.kv, self.batch, self.tree, self.q.data_ptr(), self.out.data_ptr(), self.ak, self.h, self.row, self.row,
                                     room.data_ptr(), room.numel(), scale=scale, window=window, lse_ptr=self.lse.data_ptr() if lse else 0, stream=stream)
        return room

    def seen(self, i, window):
        """[new tokens][keys] of sequence i."""
        nq, nk = self.q_len[i], max(0, self.kv_len[i])
        context = self.kv_len[i] - nq
        j = torch.arange(nk)
        pos = context + self.depths[i][:, None]
        old = (j[None] < context) & ((j[None] > pos - window) if window else True)
        new = torch.zeros(nq, nk, dtype=torch.bool)
        first = max(0, context)
        new[:, first:] = self.sees[i][:, first - context:nk - context]
        return old | new

    def expected(self, window=0, scale=0.0):
        """out, lse and each output's tolerance, in 64 bits (the terms of Step.expected)."""
        scale = scale or 1 / math.sqrt(self.d)
        rep = self.h // self.hk
        q = self.q[:, :self.h * self.d].double().cpu().view(-1, self.h, self.d)
        kt, vt = self.by_token(self.k.cpu().double()), self.by_token(self.v.cpu().double())
        out = torch.full(q.shape, 7.0, dtype=torch.float64)
        lse = torch.full(q.shape[:2], 7.0, dtype=torch.float64)
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        e = half_step(self.at)
        for i, (nq, nk) in enumerate(zip(self.q_len, self.kv_len)):
            if nq == 0:
                continue
            r = slice(self.start[i], self.start[i] + nq)
            if nk <= 0:
                out[r], lse[r] = 0, -math.inf
                continue
            s = self.slots(i)
            k, v = kt[s].nan_to_num(0, 0, 0).repeat_interleave(rep, 1), vt[s].nan_to_num(0, 0, 0).repeat_interleave(rep, 1)
            seen = self.seen(i, window)
            rows = q[r]
            a = torch.einsum("qhd,khd->hqk", rows, k) * scale
            da = torch.einsum("qhd,khd->hqk", rows.abs(), k.abs()) * abs(scale) * ((self.d + 8) * 2.0 ** -24 + (2.0 ** -20 if self.act == "f32" else 0))
            da = da.masked_fill(~seen, 0.0)
            a = a.masked_fill(~seen, -math.inf)
            l = a.logsumexp(-1)
            p = torch.where(seen, (a - torch.where(l == -math.inf, 0.0, l)[..., None]).exp(), 0.0)
            o = torch.einsum("hqk,khd->qhd", p, v)
            dp = p * (4 * da.amax(-1, keepdim=True) + 2.0 ** -20 + (e if self.act != "f32" else 2.0 ** -21)) + (2.0 ** -24 * p.amax(-1, keepdim=True) if self.act == "f16" else 0) * seen
            out[r], lse[r] = o, l.T
            tol[r] = torch.einsum("hqk,khd->qhd", dp, v.abs()) + e * o.abs() * 1.01 + 1e-30 + (nk * 2.0 ** -24) * torch.einsum("hqk,khd->qhd", p, v.abs())
            ltol[r] = (2 * da.amax(-1) + 2.0 ** -20).T + (l.abs().T.nan_to_num(0, 0, 0) + 8) * 2.0 ** -22
        return out, lse, tol, ltol


# ---- attention ------------------------------------------------------------------------

SIZES = [([1, 2, 5, 0, 26], [1, 70, 5, 9, 333]), ([17, 1, 64, 33], [17, 200, 191, 100]), ([130, 3, 65], [1000, 3, 129])]


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 4, 128), (16, 1, 128), (15, 5, 64), (40, 1, 64)])
@pytest.mark.parametrize("q_len,kv_len", SIZES)
@pytest.mark.parametrize("page,by_head", [(16, True), (24, False)])
def test_trees(gpu, act, cache, heads, kv_heads, dim, q_len, kv_len, page, by_head):
    s = Tree(q_len, kv_len, heads, kv_heads, dim, act, cache, page, by_head, seed=2, gap=16, first=2)
    s.attend()
    s.check()


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(64, 8, 128), (8, 1, 64), (32, 32, 64)])
def test_large_batches_of_trees(gpu, act, cache, heads, kv_heads, dim):
    r = np.random.RandomState(3)
    q = [int(r.randint(1, 70)) for _ in range(14)]
    kv = [n + int(r.randint(0, 900)) for n in q]
    s = Tree(q, kv, heads, kv_heads, dim, act, cache, 16, False, seed=3)
    s.attend()
    s.check()


# rows that see nothing, everything, only later tokens, only themselves; a context or none
@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,context", [(3, 0), (3, 77), (40, 0), (40, 130), (200, 0), (200, 391)])
def test_any_mask(gpu, act, cache, dim, n, context):
    r = np.random.RandomState(n + context)
    m = r.rand(n, n) < 0.3
    m[1] = np.arange(n) > 1
    m[n - 1] = True
    m[0] = False
    m[n // 2] = False
    s = Tree([n, 1], [context + n, 20], 8, 2, dim, act, cache, 16, True, seed=4, masks=[m, [[False]]])
    s.attend()
    s.check()
    if context == 0:
        assert (s.out[0] == 0).all() and (s.out[n // 2] == 0).all() and torch.isinf(s.lse[0]).all()


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 30, 64, 130, 1000])
def test_window(gpu, act, cache, dim, window):
    s = Tree([1, 40, 3, 129], [400, 300, 3, 700], 8, 2, dim, act, cache, 32, False, seed=5, near=4)
    s.attend(window=window)
    s.check(window=window)


@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32")])
def test_a_chain_is_a_tree(gpu, act, cache):
    """A chain's mask is the causal one: against the attention that has it built in, to a few roundings."""
    s = Tree([6, 70], [300, 500], 8, 2, 64, act, cache, 16, seed=6, near=1)
    s.attend()
    s.check()
    mine = s.out.clone()
    Step.attend(s)
    # both lie within the tolerance of one 64-bit result
    _, _, tol, _ = s.expected()
    assert ((mine.double() - s.out.double()).cpu()[:76, :512].view(76, 8, 64).abs() <= 2 * tol[:76]).all()


@pytest.mark.parametrize("words", [1, 2, 9])
def test_words_of_the_mask(gpu, words):
    """Fewer than the tokens need: what they do not reach is not seen. More: the rest is not looked at."""
    s = Tree([70, 5], [100, 5], 8, 2, 64, "f16", "f16", 16, seed=7, words=words)
    s.attend()
    s.check()


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim,n", [(8, 2, 64, 20), (8, 8, 128, 20), (8, 2, 64, 140), (8, 1, 128, 140)])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_values_of_unseen_tokens_do_not_reach_a_row(gpu, act, cache, heads, kv_heads, dim, n, what):
    s = Tree([n, 3], [n + 150, 30], heads, kv_heads, dim, act, cache, 16, seed=8)
    clean = Tree([n, 3], [n + 150, 30], heads, kv_heads, dim, act, cache, 16, seed=8)
    node = n // 2
    for x in (s.k, s.v):
        x[int(s.table[0, (150 + node) // 16]), (150 + node) % 16] = what
    s.attend()
    clean.attend()
    assert int(s.status.item()) == 0
    for r in range(n + 3):
        if r < n and s.sees[0][r, node]:
            assert not torch.isfinite(s.out[r].float()).any(), r
        else:
            assert torch.equal(s.out[r], clean.out[r]), r


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f32", "f16"), ("f16", "f16")])
@pytest.mark.parametrize("n", [5, 90])
def test_lengths_and_pages_that_do_not_fit(gpu, act, cache, n):
    # more new tokens than tokens: those with negative positions are nobody's keys
    s = Tree([n, 2], [n - 3, 20], 8, 2, 64, act, cache, 16, seed=9)
    s.attend()
    s.check(status=wcb.PAGED_BAD_LEN)
    assert (s.out[0:3] == 0).all() and torch.isinf(s.lse[0:3]).all()
    # a context of no tokens is nothing wrong
    s = Tree([n], [n], 8, 2, 64, act, cache, 16, seed=9)
    s.attend()
    s.check(status=0)
    # no tokens at all
    s = Tree([2], [0], 8, 2, 64, act, cache, 16, seed=9)
    s.attend()
    s.check(status=wcb.PAGED_BAD_LEN)
    # a page that is not there: its keys take no part
    s = Tree([n], [n + 100], 8, 2, 64, act, cache, 16, seed=10)
    whole = s.table.copy()
    s.table[0, 2] = s.pages
    s.upload()
    s.attend()
    assert int(s.status.item()) == wcb.PAGED_BAD_PAGE
    s.table = whole
    seen = s.seen
    s.seen = lambda i, window: seen(i, window) & (torch.arange(n + 100) // 16 != 2)
    s.check(status=wcb.PAGED_BAD_PAGE)


@pytest.mark.parametrize("start", [[0, 5, 3, 6], [-1, 2, 4, 6], [0, 2, 4, 99]])
def test_unsound_rows_are_skipped(gpu, start):
    s = Tree([2, 2, 2], [40, 20, 30], 8, 2, 64, "f16", "f16", 16, seed=11, extra=0)
    s.start = start
    s.upload()
    s.attend()
    assert int(s.status.item()) & wcb.PAGED_BAD_ROWS


def test_padded_batches_and_wrong_longest_rows(gpu):
    s = Tree([3, 70, 1], [40, 90, 7], 8, 2, 64, "f16", "f16", 16, seed=12, extra=50)
    s.batch._c.max_q_len = 1
    s.attend()
    s.check()
    s = Tree([0, 0], [5, 0], 8, 2, 64, "f16", "f16", 16, seed=12)
    s.attend()
    assert (s.out == 7.0).all()


@pytest.mark.parametrize("act,cache,n", [("f16", "f16", 5), ("f16", "f16", 60), ("f32", "f32", 60), ("f32", "f16", 20)])
def test_a_graph_follows_lengths_and_masks(gpu, act, cache, n):
    s = Tree([n, n], [300, 90], 8, 2, 64, act, cache, 16, seed=13, width=40)
    room = s.attend()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.attend(room=room, stream=torch.cuda.current_stream().cuda_stream)
    for turn, kv in enumerate(([300, 80], [n, 88], [299, n + 1])):
        t = Tree([n, n], kv, 8, 2, 64, act, cache, 16, seed=20 + turn, width=40)
        s.dev[1].copy_(torch.tensor(kv, dtype=torch.int32))
        for a, b in zip(s.tree_dev, t.tree_dev):
            a.copy_(b)
        s.kv_len, s.sees, s.depths = kv, t.sees, t.depths
        s.out.fill_(7.0)
        s.lse.fill_(7.0)
        graph.replay()
        s.check()
    assert (room[:4096] == 0).all()


@pytest.mark.parametrize("act,cache", [("bf16", "bf16"), ("f32", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("q_len", [[7], [64], [64, 3, 50]])
def test_long_contexts_and_repeatability(gpu, act, cache, q_len):
    s = Tree(q_len, [20011 + n for n in q_len], 16, 2, 128, act, cache, 64, True, seed=14)
    room = s.attend()
    s.check()
    first, lse = s.out.clone(), s.lse.clone()
    for _ in range(3):
        s.out.fill_(7.0)
        s.attend(room=room)
        assert torch.equal(first, s.out) and torch.equal(lse, s.lse)


# ---- append ---------------------------------------------------------------------------

def run_append(s, f, rot, halves, tree=None):
    g = torch.Generator().manual_seed(99)
    h, hk, d, t = s.h, s.hk, s.d, s.tokens
    width = (h + 2 * hk) * d
    qkv = torch.randn(t, width, generator=g).to(s.at).cuda()
    out = torch.full((t, h * d), 7.0, dtype=s.at, device="cuda")
    es, p = qkv.element_size(), qkv.data_ptr()
    rope = wcb.Rope(rot, halves=halves)
    f(*([s.kv, s.batch] + ([tree] if tree else []) + [rope, p, p + h * d * es, p + (h + hk) * d * es, out.data_ptr(), s.ak, h, width, width, width, h * d]))
    return qkv, out, list(rope._c.inv_freq[:rot // 2])


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("dim,rot,halves", [(64, 64, False), (128, 64, True)])
def test_append_turns_by_depth(gpu, act, cache, dim, rot, halves):
    s = Tree([1, 26, 0, 70], [1, 300, 9, 70], 8, 2, dim, act, cache, 16, True, seed=15, first=1)
    tree = wcb.PagedTree(s.tree_dev[0].data_ptr(), 0, 0)
    qkv, out, inv = run_append(s, wcb.paged_tree_append_dev, rot, halves, tree)
    x = qkv.double().cpu().view(s.tokens, 12, dim)
    ref = x.abs().amax() * 4
    kt, vt = s.by_token(s.k.double().cpu()), s.by_token(s.v.double().cpu())
    for i, (nq, nk) in enumerate(zip(s.q_len, s.kv_len)):
        r = slice(s.start[i], s.start[i] + nq)
        want = rotated(x[r, :10], nk - nq + s.depths[i], rot, halves, inv)
        got = out[r].double().cpu().view(nq, 8, dim)
        # the tolerance of append's test: f32 arithmetic on values of a few units, one rounding
        assert ((got - want[:, :8]).abs() <= half_step(s.at) * want[:, :8].abs() * 1.01 + 2.0 ** -20 * ref).all()
        sl = s.slots(i)
        gk = kt[sl][nk - nq:]
        assert ((gk - want[:, 8:]).abs() <= half_step(s.ct) * want[:, 8:].abs() * 1.01 + 2.0 ** -20 * ref).all()
        assert torch.equal(vt[sl][nk - nq:].to(s.ct), x[r, 10:].to(s.ct))
    assert (out[0] == 7.0).all() and (out[s.start[-1]:] == 7.0).all() and int(s.status.item()) == 0


def test_append_of_a_chain_is_the_chains(gpu):
    a, b = (Tree([6, 40], [1006, 40], 8, 2, 64, "f32", "f16", 16, seed=16, near=1) for _ in range(2))
    _, qa, _ = run_append(a, wcb.paged_tree_append_dev, 64, False, a.tree)
    _, qb, _ = run_append(b, wcb.paged_append_dev, 64, False)
    assert torch.equal(qa, qb)
    for x, y in ((a.k, b.k), (a.v, b.v)):
        assert torch.equal(x.nan_to_num(99.0), y.nan_to_num(99.0))


def test_append_where_there_is_no_place(gpu):
    s = Tree([3, 2], [2, 40], 8, 2, 64, "f16", "f16", 16, seed=17)
    s.table[1, 2] = s.pages
    s.upload()
    k = s.k.clone()
    run_append(s, wcb.paged_tree_append_dev, 64, False, s.tree)
    assert int(s.status.item()) == wcb.PAGED_BAD_LEN | wcb.PAGED_BAD_PAGE
    changed = (k.nan_to_num(99.0) != s.k.nan_to_num(99.0)).any(-1).any(-1)
    assert changed.sum() == 2 and changed[int(s.table[0, 0]), :2].all()


# ---- acceptance -----------------------------------------------------------------------

def accept_plain(start, parent, token, sampled, max_path):
    paths, tokens, counts = [], [], []
    for lo, hi in zip(start, start[1:]):
        way, out, at = [], [], 0
        while lo + at < hi and len(way) < max_path:
            way.append(at)
            out.append(int(sampled[lo + at]))
            nxt = [i for i in range(at + 1, hi - lo) if parent[lo + i] == at and token[lo + i] == out[-1] >= 0]
            if not nxt:
                break
            at = nxt[0]
        counts.append(len(way))
        paths.append(way + [-1] * (max_path - len(way)))
        tokens.append(out + [-1] * (max_path - len(way)))
    return paths, tokens, counts


def run_accept(start, parent, token, sampled, max_path, extra=2):
    dev = [torch.tensor(np.asarray(x), dtype=torch.int32).cuda() for x in (start, [0] * (len(start) - 1), parent, token, sampled)]
    n = len(start) - 1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = [torch.full((n + 1, max_path), 77, dtype=torch.int32, device="cuda") for _ in range(2)] + [torch.full((n + 1,), 77, dtype=torch.int32, device="cuda")]
    batch = wcb.PagedBatch(dev[0].data_ptr(), dev[1].data_ptr(), dev[1].data_ptr(), n, len(parent), 1, 1, status.data_ptr())
    wcb.tree_accept_dev(batch, dev[2].data_ptr(), dev[3].data_ptr(), dev[4].data_ptr(), max_path, *[x.data_ptr() for x in out])
    assert all((x[n] == 77).all() for x in out)
    return [x[:n].tolist() for x in out], int(status.item())


@pytest.mark.parametrize("sizes", [[1], [26], [0, 3, 1, 0, 64], [200] * 40, [5000, 2], [4096, 4097]])
@pytest.mark.parametrize("max_path", [1, 4, 300])
def test_accept(gpu, sizes, max_path):
    rng = np.random.RandomState(len(sizes) + max_path)
    start, parent = [2], [7, -9]  # rows before the first sequence
    for n in sizes:
        parent += random_tree(rng, n) if n else []
        start.append(start[-1] + n)
    parent += [3, 3]
    token = rng.randint(0, 3, len(parent))  # siblings with one token among them
    sampled = rng.randint(-1, 3, len(parent))
    got, status = run_accept(start, parent, token, sampled, max_path)
    want = accept_plain(start, parent, token, sampled, max_path)
    assert list(got) == [list(x) for x in want] and status == 0
    assert max_path < 4 or len(sizes) < 20 or max(want[2]) >= 3


def test_accept_the_whole_of_a_chain(gpu):
    n = 6000
    got, status = run_accept([0, n], [-1] + list(range(n - 1)), [(i * 7) % 100 for i in range(n)], [((i + 1) * 7) % 100 for i in range(n)], n + 3)
    assert got[0][0] == list(range(n)) + [-1] * 3 and got[2] == [n] and status == 0


def test_accept_reports_parents_that_come_later(gpu):
    got, status = run_accept([0, 4], [-1, 2, 0, 3], [5, 5, 5, 5], [5, 5, 5, 5], 4)
    assert got[0][0] == [0, 2, -1, -1] and status == wcb.PAGED_BAD_TREE
    got, status = run_accept([0, 3], [9, 0, -1], [5, 5, 5], [5, 5, 5], 4)  # the root's is not read; -1: no one's child
    assert got[0][0] == [0, 1, -1, -1] and status == 0
    got, status = run_accept([0, 5, 3], [-1, 0, 0], [5, 5, 5], [5, 5, 5], 2)
    assert status & wcb.PAGED_BAD_ROWS and got[2] == [0, 0] and got[0] == [[-1, -1], [-1, -1]]


# ---- keep -----------------------------------------------------------------------------

class Layers:
    def __init__(self, q_len, kv_len, layers=3, first=0, **o):
        self.steps = [Step(q_len, kv_len, seed=50 + i, first=first, **o) for i in range(layers)]
        for s in self.steps[1:]:
            s.table = self.steps[0].table
        self.s = self.steps[0]

    def keep(self, paths, counts=None, max_path=None, stream=0):
        counts = counts or [len(p) for p in paths]
        m = max_path or max(max(len(p) for p in paths), 1)
        path = torch.full((len(paths), m), -5, dtype=torch.int32)
        for i, p in enumerate(paths):
            path[i, :len(p)] = torch.tensor(p[:m], dtype=torch.int32)
        self.dev = [path.cuda(), torch.tensor(counts, dtype=torch.int32).cuda()]
        wcb.paged_keep_dev(wcb.PagedLayers([s.kv for s in self.steps]), self.s.batch, self.dev[0].data_ptr(), m, self.dev[1].data_ptr(), stream=stream)

    def run_and_check(self, paths, skipped=(), status=0, **o):
        """Moves, and nothing but the moves, bit by bit. skipped: (sequence, i) that do not move."""
        want = []
        for s in self.steps:
            for pool in (s.k, s.v):
                w = s.by_token(pool.clone()).t
                for q, p in enumerate(paths):
                    context = s.kv_len[q] - s.q_len[q]
                    place = [(int(s.table[q, (context + j) // s.page]), (context + j) % s.page) if 0 <= (context + j) // s.page < s.table.shape[1] else None for j in range(s.q_len[q])]
                    old = w.clone()
                    for i, j in enumerate(p):
                        if (q, i) not in skipped:
                            w[place[i]] = old[place[j]]
                want.append(w)
        self.keep(paths, **o)
        torch.cuda.synchronize()
        got = [s.by_token(pool).t for s in self.steps for pool in (s.k, s.v)]
        bits = torch.int32 if got[0].element_size() == 4 else torch.int16
        for g, w in zip(got, want):
            assert torch.equal(g.contiguous().view(bits), w.contiguous().view(bits))
        assert int(self.s.status.item()) == status


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv_heads,dim,page,by_head", [(2, 64, 16, False), (8, 128, 24, True), (5, 64, 1, False), (40, 128, 64, True)])
def test_keep(gpu, cache, kv_heads, dim, page, by_head):
    x = Layers([26, 1, 0, 9, 70], [333, 5, 9, 9, 100], heads=kv_heads, kv_heads=kv_heads, dim=dim, act="f32", cache=cache, page=page, by_head=by_head, first=2)
    x.run_and_check([[0, 3, 4, 17, 25], [0], [], [0, 1, 2], [1, 2, 4, 8, 16, 32, 33, 34, 35, 36, 69]])


def test_keep_long_paths(gpu):
    n = 700
    rng = np.random.RandomState(1)
    paths = [sorted(rng.choice(n, 300, replace=False).tolist()), list(range(1, n)), list(range(n)), [n - 1]]
    Layers([n] * 4, [n + 5, n, n + 64, n + 1], heads=2, kv_heads=2, dim=64, act="f32", cache="f16", page=16).run_and_check(paths)


def test_keep_many_layers(gpu):
    Layers([5, 6], [40, 6], layers=131, heads=2, kv_heads=1, dim=64, act="f32", cache="f16", page=8).run_and_check([[0, 2, 4], [3]])


def test_keep_what_it_does_not_follow(gpu):
    o = dict(layers=2, heads=2, kv_heads=2, dim=64, act="f32", cache="f16", page=16)
    for bad in ([0, 3, 3], [0, 4, 2], [0, 5], [-1, 2], [0, 1 << 30]):
        x = Layers([5, 5], [40, 20], **o)
        x.run_and_check([bad, [0, 4]], skipped=[(0, i) for i in range(3)], status=wcb.PAGED_BAD_TREE)
    # counts are held to the path's room; what lies behind it is not read
    x = Layers([5, 5], [40, 20], **o)
    x.run_and_check([[1, 2], [0, 4]], counts=[9, 2])
    x = Layers([5, 5], [40, 20], **o)
    x.run_and_check([[], [0, 4]], counts=[-3, 2])
    # positions below zero, pages that are not there
    x = Layers([5, 5], [3, 20], **o)
    x.run_and_check([[0, 3, 4], [0, 4]], skipped=[(0, 0), (0, 1)], status=wcb.PAGED_BAD_LEN)
    x = Layers([20, 5], [40, 20], **o)
    for s in x.steps:
        s.table = s.table.copy()
    x.s.table[0, 2] = -1
    x.s.upload()
    x.run_and_check([[5, 11, 12, 13], [0, 4]], skipped=[(0, 2), (0, 3)], status=wcb.PAGED_BAD_PAGE)


# ---- the steps of a serving loop --------------------------------------------------------

@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("bf16", "bf16"), ("f32", "f32")])
def test_steps_with_trees(gpu, act, cache):
    """Append, attend, sample, accept, keep for a ragged batch of trees in two layers, captured as one graph and replayed: what
    comes out is what the tokens accepted so far, as plain sequences, give."""
    h, hk, d, v, layers, n = 8, 2, 64, 50, 2, 12
    q_len = [n, 1, 7]
    steps = [Tree(q_len, [200, 160, 180], h, hk, d, act, cache, 16, True, seed=60, extra=1) for _ in range(layers)]  # pages for the tokens to come
    s = steps[0]
    for x in steps:
        x.kv_len = [54 + n, 12, 7]
        x.upload()
    g = torch.Generator(device="cuda").manual_seed(61)
    rng = np.random.RandomState(62)
    t, width = s.tokens, (h + 2 * hk) * d
    emb = torch.randn(layers, v, width, generator=g, device="cuda").to(s.at)  # a token's projections: by its id alone
    wout = torch.randn(layers * h * d, v, generator=g, device="cuda") * 0.2
    draft = torch.zeros(t, dtype=torch.int32, device="cuda")
    parent = torch.zeros(t, dtype=torch.int32, device="cuda")
    qkv = torch.empty(layers, t, width, dtype=s.at, device="cuda")
    q = torch.empty(layers, t, h * d, dtype=s.at, device="cuda")
    logits, probs = torch.empty(t, v, device="cuda"), torch.empty(t, v, device="cuda")
    u = torch.empty(t, device="cuda")
    temp, top_k = torch.full((t,), 0.8, device="cuda"), torch.full((t,), 20, dtype=torch.int32, device="cuda")
    sampled = torch.empty(t, dtype=torch.int32, device="cuda")
    path, out = (torch.empty(3, n, dtype=torch.int32, device="cuda") for _ in range(2))
    count = torch.empty(3, dtype=torch.int32, device="cuda")
    rope, room = wcb.Rope(d), s.workspace()
    es = qkv.element_size()
    all_layers = wcb.PagedLayers([x.kv for x in steps])
    settings = wcb.Sampling(temp.data_ptr(), top_k.data_ptr())

    def step():
        st = torch.cuda.current_stream().cuda_stream
        for i, x in enumerate(steps):
            qkv[i].copy_(emb[i][draft.long()])
            p = qkv[i].data_ptr()
            wcb.paged_tree_append_dev(x.kv, s.batch, s.tree, rope, p, p + es * h * d, p + es * (h + hk) * d, q[i].data_ptr(), s.ak, h, width, width, width, h * d, stream=st)
            wcb.paged_tree_attention_dev(x.kv, s.batch, s.tree, q[i].data_ptr(), x.out.data_ptr(), s.ak, h, h * d, s.row, room.data_ptr(), room.numel(), stream=st)
        logits.copy_(torch.cat([x.out.float() for x in steps], -1) @ wout)
        wcb.sample_dev(logits.data_ptr(), wcb.KV_F32, t, v, settings, u.data_ptr(), sampled.data_ptr(), probs_ptr=probs.data_ptr(), stream=st)
        wcb.tree_accept_dev(s.batch, parent.data_ptr(), draft.data_ptr(), sampled.data_ptr(), n, path.data_ptr(), out.data_ptr(), count.data_ptr(), stream=st)
        wcb.paged_keep_dev(all_layers, s.batch, path.data_ptr(), n, count.data_ptr(), stream=st)

    history = [[] for _ in q_len]  # the tokens in the cache behind the first context
    base = [k - m for k, m in zip(s.kv_len, q_len)]
    step()  # warm; leaves rows that the next step writes again
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    accepted = 0
    last = [3, 4, 5]
    for turn in range(4):
        tree = Tree(q_len, s.kv_len, h, hk, d, act, cache, 16, True, seed=70 + turn, extra=1)
        par = [p for one in tree.parent for p in one] + [-1]
        ids = rng.randint(0, v, t)
        for i, first in enumerate(s.start[:-1]):
            ids[first] = last[i]
        for a, b in zip(s.tree_dev, tree.tree_dev):
            a.copy_(b)
        parent.copy_(torch.tensor(par, dtype=torch.int32))
        u.copy_(torch.rand(t, generator=g, device="cuda"))
        s.dev[1].copy_(torch.tensor(s.kv_len, dtype=torch.int32))
        # drafts that the target takes now and then: a first run tells what it samples
        draft.copy_(torch.tensor(ids, dtype=torch.int32))
        # the tree is grown level by level from what the target samples at its nodes, half of the time
        before = [(x.k.clone(), x.v.clone()) for x in steps]
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            got = sampled.tolist()
            for i, first in enumerate(s.start[:-1]):
                for j in range(1, q_len[i]):
                    if rng.rand() < 0.6:
                        ids[first + j] = got[first + par[first + j]]
            draft.copy_(torch.tensor(ids, dtype=torch.int32))
            for x, (k, vv) in zip(steps, before):
                x.k.copy_(k)
                x.v.copy_(vv)
        graph.replay()
        torch.cuda.synchronize()
        # sampling and acceptance by themselves
        toks, ps = sample_plain(logits.cpu().double().numpy(), [0.8] * t, [20] * t, [1.0] * t, [0.0] * t, u.cpu().double().numpy())
        assert sampled.tolist() == toks and np.abs(probs.cpu().numpy() - ps).max() <= 2.0 ** -23
        want = accept_plain(s.start, par, ids, sampled.tolist(), n)
        assert path.tolist() == want[0] and out.tolist() == want[1] and count.tolist() == want[2]
        accepted += sum(want[2]) - 3
        # the accepted tokens' rows of the cache, and the outputs at their nodes, as a plain sequence gives them
        for i in range(3):
            way = want[0][i][:want[2][i]]
            new = [int(ids[s.start[i] + j]) for j in way]
            m = base[i] + len(history[i])
            for li, x in enumerate(steps):
                sl = x.slots(i)
                keys, vals = x.by_token(x.k.double().cpu())[sl], x.by_token(x.v.double().cpu())[sl]
                proj = emb[li].double().cpu()[new].view(len(new), h + 2 * hk, d)
                pos = torch.arange(m, m + len(new))
                turned = rotated(proj[:, :h + hk], pos, d, False, list(rope._c.inv_freq[:d // 2]))
                tol = half_step(s.ct) * 1.01 + 2.0 ** -18
                assert ((keys[m:m + len(new)] - turned[:, h:]).abs() <= tol * turned[:, h:].abs().clamp(min=1.0)).all()
                assert torch.equal(vals[m:m + len(new)].to(s.ct), proj[:, h + hk:].to(s.ct))
                if i == 1:
                    continue
                # keys in the cache are rounded already; the queries once
                qq = turned[:, :h].to(s.at).double()
                kk, vv = keys[:m + len(new)].repeat_interleave(h // hk, 1), vals[:m + len(new)].repeat_interleave(h // hk, 1)
                a = torch.einsum("qhd,khd->hqk", qq, kk) / 8
                a = a.masked_fill(torch.arange(m + len(new))[None, :] > pos[:, None], -math.inf)
                o = torch.einsum("hqk,khd->qhd", a.softmax(-1), vv)
                rows = x.out[[s.start[i] + j for j in way]].double().cpu().view(len(way), h, d)
                # queries that differ by their own rounding (scores of up to 8 units: 8 half steps of p), p and o rounded
                assert (rows - o).abs().max() <= (24 * half_step(s.at) + 2.0 ** -16) * vv.abs().max()
            history[i] += new
            last[i] = want[1][i][want[2][i] - 1]
        s.kv_len = [b + len(x) + m for b, x, m in zip(base, history, q_len)]
        for x in steps:
            x.kv_len = s.kv_len
    assert accepted >= 4 and int(s.status.item()) == 0


# ---- calls side by side -----------------------------------------------------------------

def test_trees_and_chains_share_a_workspace(gpu):
    a = Tree([40, 3], [3000, 500], 8, 2, 128, "f16", "f16", 16, seed=80)
    b = Step([4, 1, 200], [900, 2500, 800], 8, 2, 128, "f16", "f16", 16, seed=81)
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
    assert (room[:4096] == 0).all()


def test_two_streams(gpu):
    s = [Tree([30, 1, 64], [3000, 500, 900], 8, 2, 64, *pair, 16, seed=82 + i) for i, pair in enumerate([("f16", "f16"), ("f32", "f32")])]
    rooms, streams = [x.workspace() for x in s], [torch.cuda.Stream() for _ in s]
    torch.cuda.synchronize()
    for _ in range(10):
        for x, r, st in zip(s, rooms, streams):
            x.attend(room=r, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for x in s:
        x.check()


def _run(code, env=None):
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = code.format(pkg=os.path.join(os.path.dirname(here), "wasm-chord_b200"), tests=here)
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=dict(os.environ, **(env or {})))


FIRST_CALLS = """
import sys
sys.path.insert(0, {pkg!r}); sys.path.insert(0, {tests!r})
import torch, wcb, numpy as np
import test_gpu_tree as t
for act, cache in t.PAIRS:
    for q_len in ([5, 2], [90, 3]):
        s = t.Tree(q_len, [300, 40], 8, 2, 64, act, cache, 16, seed=40)
        room, graph = s.workspace(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.attend(room=room, stream=torch.cuda.current_stream().cuda_stream)
        graph.replay()
        graph.replay()
        s.check()
from test_gpu_sample import sample_plain, KIND
for kind in KIND:
    for n, v in ((2, 5000), (1, 900001)):
        l = torch.randn(n, v, device="cuda").to(KIND[kind][0])
        u, out, p = torch.rand(n, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda"), torch.full((n,), 0.9, device="cuda")
        settings, graph = wcb.Sampling(0, 0, p.data_ptr(), 0), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            wcb.sample_dev(l.data_ptr(), KIND[kind][1], n, v, settings, u.data_ptr(), out.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
        graph.replay()
        assert out.tolist() == sample_plain(l.double().cpu().numpy(), [1.0] * n, [0] * n, [float(p[0])] * n, [0.0] * n, u.double().cpu().numpy())[0]
print("captured first")
"""


def test_the_first_calls_may_be_captured_ones(gpu):
    r = _run(FIRST_CALLS)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]


WAITS = """
import sys
sys.path.insert(0, {pkg!r}); sys.path.insert(0, {tests!r})
import time, torch, wcb
import test_gpu_tree as t
for act, cache in (("bf16", "bf16"), ("f16", "f16"), ("f32", "f16")):
    for dim in (64, 128):
        for q, kv in (([200], [2000]), ([5, 1, 2], [700, 65, 900]), ([1, 70, 64], [700, 1000, 230])):
            s = t.Tree(q, kv, 8, 2, dim, act, cache, 64, seed=70)
            torch.cuda.synchronize()
            begin = time.time()
            s.attend()
            torch.cuda.synchronize()
            assert time.time() - begin < 2, time.time() - begin
            assert int(s.status.item()) & wcb.PAGED_ABORTED, (act, cache, dim, q)
# what brings nothing by bulk copy works as ever: an f32 cache on the tensor cores
s = t.Tree([200], [900], 8, 2, 64, "f32", "f32", 16, seed=71)
s.attend()
s.check()
print("every wait ended")
"""


def test_waits_end(gpu):
    """Copies that do not come (test_gpu_paged_waits.py): each wait runs out, the call says so, the device stays usable."""
    r = _run(WAITS, {"WCB_TEST_WITHHOLD_COPY": "1"})
    assert r.returncode == 0 and "every wait ended" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]
