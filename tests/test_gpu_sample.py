"""Sampling rows of logits on the GPU (wcb_sample_dev) against a plain 64-bit form."""
import numpy as np
import pytest

import wcb

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

KIND = {"f32": (torch.float32, wcb.KV_F32), "f16": (torch.float16, wcb.KV_F16), "bf16": (torch.bfloat16, wcb.KV_BF16)}


def kept_plain(l, t, k, p, m):
    """Weights of one row (64 bits), zero where not kept; None without candidates."""
    some = ~(np.isnan(l) | (l == -np.inf))
    if not some.any():
        return None
    top = l[some].max()
    t = float(np.float32(t))
    order = sorted(np.flatnonzero(some).tolist(), key=lambda j: (-l[j], j)) if some.sum() < 3000 else [j for j in np.argsort(-np.where(some, l, -np.inf), kind="stable").tolist() if some[j]]
    with np.errstate(invalid="ignore", over="ignore"):
        x = np.where(l == top, 0.0, (l - top) / t) if t > 0 and top < np.inf else np.where(l == top, 0.0, -np.inf)
        e = np.where(some & ~np.isnan(x), np.exp(np.where(some, x, -np.inf)), 0.0)
    if not t > 0:
        k, p, m = 1, 1.0, 0.0
    if k > 0:
        order = order[:k]
    p, m = float(np.float32(p)), float(np.float32(m))
    if p < 1:
        w = e[order]
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = int((before < max(p, 0.0) * w.sum()).sum())
        order = order[:max(n, 1)]
    if m > 0:
        order = [j for j in order if e[j] >= min(m, 1.0)]
    w = np.zeros_like(e)
    w[order] = e[order]
    return w


def sample_plain(l, t, k, p, m, u):
    tokens, probs = [], np.zeros(l.shape)
    for i in range(len(l)):
        w = kept_plain(l[i], t[i], k[i], p[i], m[i])
        if w is None:
            tokens.append(-1)
            continue
        x = min(max(u[i], 0.0), 0.99999994) if u[i] == u[i] else 0.0
        c = np.cumsum(w)
        tokens.append(int(np.searchsorted(c, x * c[-1], side="right")))
        probs[i] = w / c[-1]
    return tokens, probs


def run(l, kind="f32", t=None, k=None, p=None, m=None, u=None, probs=True, pad=0, stream=0):
    n, v = l.shape
    ct, ck = KIND[kind]
    rows = torch.full((n, v + pad), 1e4, dtype=ct, device="cuda")
    rows[:, :v] = torch.as_tensor(l).to(ct).cuda()
    put = lambda x, dt: torch.tensor(x, dtype=dt, device="cuda") if x is not None else None
    dev = [put(t, torch.float32), put(k, torch.int32), put(p, torch.float32), put(m, torch.float32)]
    u = np.random.RandomState(0).rand(n) if u is None else u
    du = put(list(u), torch.float32)
    tokens = torch.full((n + 1,), 77, dtype=torch.int32, device="cuda")
    pr = torch.full((n, v + pad), 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    s = wcb.Sampling(*[x.data_ptr() if x is not None else 0 for x in dev])
    wcb.sample_dev(rows.data_ptr(), ck, n, v, s, du.data_ptr(), tokens.data_ptr(), row_stride=v + pad, probs_ptr=pr.data_ptr() if probs else 0, probs_stride=v + pad,
                   status_ptr=status.data_ptr(), stream=stream)
    torch.cuda.synchronize()
    assert tokens[n] == 77
    if probs and pad:
        assert (pr[:, v:] == 7.0).all()
    return tokens[:n].tolist(), pr[:, :v].cpu().double().numpy(), int(status.item()), rows[:, :v].cpu().double().numpy(), du.cpu().double().numpy()


def check(l, kind="f32", t=None, k=None, p=None, m=None, u=None, pad=0, status=0):
    n, v = l.shape
    got, probs, st, exact, du = run(l, kind, t, k, p, m, u, True, pad)
    want, ps = sample_plain(exact, t or [1.0] * n, k or [0] * n, p or [1.0] * n, m or [0.0] * n, du)
    assert st == status
    # the same tokens are kept; f32 rounding, weights of 64 bits whose sum is rounded to steps of 2^-43 (and below 2^-60 none)
    assert ((probs > 0) == (ps > 2.0 ** -59)).all() or (ps[(probs > 0) != (ps > 0)] < 2.0 ** -59).all()
    assert (np.abs(probs - ps) <= ps * (2.0 ** -24 + 2.0 ** -40 + v * 2.0 ** -44) + 2.0 ** -59).all()
    for i in range(n):
        if got[i] == want[i]:
            continue
        # a draw within the sums' rounding of a border: half a step of 2^-43 of the largest weight for each token
        c = np.cumsum(ps[i])
        x = min(max(du[i], 0.0), 0.99999994)
        assert ps[i, got[i]] > 0 and abs(c[min(got[i], want[i])] - x) <= v * 2.0 ** -43, (i, got[i], want[i])
    # the same without the probabilities
    assert run(l, kind, t, k, p, m, u, False, pad)[0] == got
    return got, probs


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (0.8, 1, 1.0, 0.0), (1.0, 0, 0.95, 0.0), (1.5, 0, 0.3, 0.0), (1.0, 0, 1.0, 0.05),
            (0.6, 20, 0.95, 0.3), (2.0, 900, 0.99, 0.001), (1.0, 7, 0.5, 0.0), (0.1, 50, 0.9, 0.0), (50.0, 0, 0.5, 0.0), (1.0, 1 << 30, 1.0, 1.0), (1.0, 0, 0.0, 0.0)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("v,pad", [(1, 0), (2, 1), (31, 0), (33, 3), (257, 0), (1000, 7), (2049, 0), (32000, 0), (50257, 5)])
def test_settings(gpu, kind, v, pad):
    r = np.random.RandomState(v)
    n = len(SETTINGS)
    l = r.randn(n, v) * 3
    t, k, p, m = (list(x) for x in zip(*SETTINGS))
    check(l, kind, t, k, p, m, r.rand(n).tolist(), pad)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n,v", [(1, 100003), (3, 131072), (40, 100003), (300, 5003), (2, 1 << 20)])
@pytest.mark.parametrize("setting", [(0.9, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (1.0, 5000, 0.97, 0.001)])
def test_sizes(gpu, kind, n, v, setting):
    if v == 1 << 20 and kind == "bf16":
        n = 1
    r = np.random.RandomState(n)
    check(r.randn(n, v).astype(np.float32) * 2.5, kind, *([x] * n for x in setting), r.rand(n).tolist())


# equal logits, among which the lowest indices are kept
@pytest.mark.parametrize("v", [5, 64, 1000, 40000])
@pytest.mark.parametrize("levels", [1, 2, 5])
def test_ties(gpu, v, levels):
    r = np.random.RandomState(v + levels)
    n = 12
    l = r.randint(0, levels, (n, v)).astype(np.float32) * 0.5
    k = [0, 1, 3, v // 2, v - 1, v, 0, 0, 0, 4, v // 3 + 1, 0]
    p = [1.0] * 6 + [0.5, 0.25, 0.875, 0.5, 0.5, 2.0 ** -20]
    check(l, "f32", [1.0] * n, [max(x, 0) for x in k], p, [0.0] * n, r.rand(n).tolist())


def test_exact_halves(gpu):
    # 8 equal logits: the sum before the fifth is half of all, which is not less than half
    l = np.zeros((3, 8), np.float32)
    _, probs = check(l, "f32", [1.0] * 3, [0, 6, 0], [0.5, 0.5, 0.625], [0.0] * 3, [0.0, 0.99, 0.99])
    assert (probs[0] > 0).sum() == 4 and (probs[1] > 0).sum() == 3 and (probs[2] > 0).sum() == 5
    # weights of 1 and 1 / 2 by a temperature: min-p at the border keeps them, above it does not
    l = np.array([[0.0, 1.0, -1.0]] * 2, np.float32)
    check(l, "f32", [1.0, 1.0], [0, 0], [1.0, 1.0], [0.36, 0.37], [0.9, 0.9])


def test_draws_at_the_ends(gpu):
    l = np.tile(np.array([-np.inf, 0.0, 0.0, -np.inf, 1.0, np.nan], np.float32), (7, 1))
    got, _ = check(l, "f32", u=[0.0, 1.0, 2.0, -1.0, float("nan"), 0.99999994, float("inf")])
    assert got[0] == got[3] == got[4] == 1 and got[1] == got[2] == got[5] == got[6] == 4


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("v", [6, 3001])
def test_infinities_and_nan(gpu, kind, v):
    r = np.random.RandomState(v)
    l = r.randn(8, v) * 2
    l[0] = np.nan
    l[1] = -np.inf
    l[2, ::2] = np.nan
    l[3, ::3] = -np.inf
    l[4, [1, 4]] = np.inf
    l[5] = -np.inf
    l[5, v - 1] = -60000.0
    l[6, 1:] = torch.finfo(KIND[kind][0]).min  # a mask's lowest value
    l[7] = torch.finfo(KIND[kind][0]).min
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 4, 0.9, 0.1), (1.0, 0, 0.7, 0.0)):
        got, probs = check(l, kind, [t] * 8, [k] * 8, [p] * 8, [m] * 8, [0.6] * 8, status=wcb.PAGED_BAD_PROBS)
        assert got[:2] == [-1, -1] and (probs[:2] == 0).all() and got[4] in (1, 4) and got[5] == v - 1 and got[6] == 0


def test_temperatures_of_any_size(gpu):
    r = np.random.RandomState(1)
    t = [1e-45, 1e-30, 1e-3, 1e3, 1e30, float("inf"), -1.0, float("nan"), 0.0, -0.0]
    l = np.tile((r.randn(1, 500) * 3).astype(np.float32), (len(t), 1))
    got, probs = check(l, "f32", t, u=[0.5] * len(t))
    best = int(l[0].argmax())
    assert [got[i] for i in (0, 1, 6, 7, 8, 9)] == [best] * 6
    # settings that are no numbers are off
    check(l[:2], "f32", [1.0] * 2, [-5, 0], [float("nan"), 7.0], [float("nan"), -1.0], [0.5] * 2)


def test_signed_zeros_are_equal(gpu):
    l = np.array([[-1.0, -0.0, 0.0, -0.0]] * 3, np.float32)
    got, probs = check(l, "f32", [0.0, 1.0, 1.0], [0, 2, 0], [1.0, 1.0, 0.3], u=[0.5, 0.99, 0.5])
    # the third: 0.3 of 3 + e^-1 is 1.01, more than the one before the second zero; half of the two that are kept is the first, which has to be exceeded
    assert got == [1, 2, 2]


def test_no_settings_and_a_row_at_a_time(gpu):
    r = np.random.RandomState(2)
    l = r.randn(9, 1234).astype(np.float32)
    got, _ = check(l)
    rows = torch.tensor(l, device="cuda")
    u = torch.tensor(np.random.RandomState(0).rand(9), dtype=torch.float32, device="cuda")
    out = torch.full((9,), 77, dtype=torch.int32, device="cuda")
    for i in range(9):
        wcb.sample_dev(rows[i].data_ptr(), wcb.KV_F32, 1, 1234, None, u[i:].data_ptr(), out[i:].data_ptr())
    assert out.tolist() == got


def test_frequencies(gpu):
    # 40000 draws of 6 tokens: each count within 6 standard deviations
    n = 40000
    l = np.tile(np.array([0.0, 1.0, -1.0, 2.0, 0.5, -3.0], np.float32), (n, 1))
    got, *_ = run(l, t=[0.9] * n, p=[0.98] * n, u=np.random.RandomState(5).rand(n), probs=False)
    w = kept_plain(l[0].astype(np.float64), 0.9, 0, 0.98, 0.0)
    w /= w.sum()
    c = np.bincount(got, minlength=6)
    assert (np.abs(c - n * w) <= 6 * np.sqrt(n * w * (1 - w)) + 1e-9).all()


def test_a_graph_follows_settings_and_logits(gpu):
    n, v = 5, 4099
    rows, u = torch.empty(n, v, device="cuda"), torch.empty(n, device="cuda")
    t, k, p, m = torch.ones(n, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")
    out = torch.empty(n, dtype=torch.int32, device="cuda")
    s = wcb.Sampling(t.data_ptr(), k.data_ptr(), p.data_ptr(), m.data_ptr())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        wcb.sample_dev(rows.data_ptr(), wcb.KV_F32, n, v, s, u.data_ptr(), out.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    g = torch.Generator(device="cuda").manual_seed(3)
    for ks, ps in ((0, 1.0), (10, 1.0), (0, 0.6), (2000, 0.9)):
        rows.copy_(torch.randn(n, v, generator=g, device="cuda") * 2)
        u.copy_(torch.rand(n, generator=g, device="cuda"))
        k.fill_(ks)
        p.fill_(ps)
        graph.replay()
        torch.cuda.synchronize()
        want, _ = sample_plain(rows.double().cpu().numpy(), [1.0] * n, [ks] * n, [float(p[0])] * n, [0.0] * n, u.double().cpu().numpy())
        assert out.tolist() == want


def test_two_calls_at_once(gpu):
    r = np.random.RandomState(4)
    l = [torch.tensor(r.randn(64, 20011) * 2, dtype=torch.float32, device="cuda") for _ in range(2)]
    u = torch.rand(64, device="cuda")
    p = torch.full((64,), 0.9, device="cuda")
    s = wcb.Sampling(0, 0, p.data_ptr(), 0)
    alone = [torch.empty(64, dtype=torch.int32, device="cuda") for _ in range(2)]
    for x, o in zip(l, alone):
        wcb.sample_dev(x.data_ptr(), wcb.KV_F32, 64, 20011, s, u.data_ptr(), o.data_ptr())
    torch.cuda.synchronize()
    streams, both = [torch.cuda.Stream() for _ in range(2)], [torch.empty(64, dtype=torch.int32, device="cuda") for _ in range(2)]
    for _ in range(5):
        for x, o, st in zip(l, both, streams):
            wcb.sample_dev(x.data_ptr(), wcb.KV_F32, 64, 20011, s, u.data_ptr(), o.data_ptr(), stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, both))


# more equal logits than a list holds: found over the whole row, by one CTA a row (300 rows) and by eight (3 rows); fewer: in the list
@pytest.mark.parametrize("n,v", [(300, 9001), (3, 70001), (300, 700), (3, 20000)])
@pytest.mark.parametrize("step", [0.0, 0.25])
def test_many_equal_logits(gpu, n, v, step):
    r = np.random.RandomState(n + v)
    l = np.floor(r.rand(n, v) * 6).astype(np.float32) * step
    kinds = [(1.0, 0, 0.5, 0.0), (0.7, v // 3, 1.0, 0.0), (1.0, v // 2, 0.9, 0.0), (0.5, v - 1, 0.99, 0.2), (1.0, 33, 0.7, 0.0), (1.0, 0, 2.0 ** -10, 0.0)]
    t, k, p, m = (list(x) for x in zip(*[kinds[i % len(kinds)] for i in range(n)]))
    check(l, "f32", t, k, p, m, r.rand(n).tolist())


# logits far from zero, temperatures so low that a bin is no more than their rounding: without bins
@pytest.mark.parametrize("offset,t", [(1e5, 1.0), (-3e6, 50.0), (0.0, 1e-3), (2000.0, 0.3)])
@pytest.mark.parametrize("v", [500, 30001])
def test_logits_far_from_zero(gpu, offset, t, v):
    r = np.random.RandomState(v)
    l = (r.randn(6, v) * 2.5 + offset).astype(np.float32)
    check(l, "f32", [t] * 6, [0, 40, 0, 900, 0, 5], [0.9, 1.0, 1.0, 0.95, 0.3, 0.5], [0.0, 0.0, 0.05, 0.0, 0.01, 0.0], r.rand(6).tolist())


def test_flat_rows(gpu):
    # next to no differences: every weight counts
    r = np.random.RandomState(3)
    l = (r.randn(4, 131072) * 0.05).astype(np.float32)
    check(l, "f32", [1.0, 2.0, 0.7, 1.0], [0, 0, 100000, 50], [0.9, 0.99, 0.5, 1.0], [0.0] * 4, r.rand(4).tolist())


def test_rows_far_apart(gpu):
    # offsets past 32 bits: the second row begins 5 GB behind the first (of one buffer)
    v, stride = 1001, 1_300_000_000
    if torch.cuda.mem_get_info()[0] < 12e9:
        pytest.skip("needs 11 GB")
    rows = torch.empty(2 * stride, dtype=torch.float32, device="cuda")
    r = np.random.RandomState(4)
    l = r.randn(2, v).astype(np.float32)
    for i in range(2):
        rows[i * stride:i * stride + v] = torch.tensor(l[i], device="cuda")
    u = torch.tensor([0.3, 0.8], device="cuda")
    out = torch.empty(2, dtype=torch.int32, device="cuda")
    wcb.sample_dev(rows.data_ptr(), wcb.KV_F32, 2, v, None, u.data_ptr(), out.data_ptr(), row_stride=stride)
    assert out.tolist() == sample_plain(l.astype(np.float64), [1.0] * 2, [0] * 2, [1.0] * 2, [0.0] * 2, u.double().cpu().numpy())[0]


# more rows than run at once are taken in an order of their own: each is done once, whatever its settings
@pytest.mark.parametrize("n", [297, 700, 2048, 2049])
@pytest.mark.parametrize("given", ["all", "top_p", "top_k", "temperature"])
def test_many_rows_of_many_kinds(gpu, n, given):
    r = np.random.RandomState(n)
    rows = [SETTINGS[i] for i in r.randint(0, len(SETTINGS), n)]
    t, k, p, m = (list(x) for x in zip(*rows))
    if given != "all":
        t, k, p, m = (x if given == name else None for x, name in ((t, "temperature"), (k, "top_k"), (p, "top_p"), (m, "min_p")))
    check(r.randn(n, 211) * 3, "f32", t, k, p, m, r.rand(n).tolist())
