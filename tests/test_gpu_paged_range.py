"""Paged attention over numbers of very different sizes: large finite keys and values that a row does not see or
gives no weight, a key that takes most of the weight, and the low-order parts of f32 numbers. Held to bounds near the
kernels' own errors, row by row, against 64 bits.

Bound for f32 activations. Each weight p_j carries a relative error of its score's error, of the exponential and
of the splits and short sums: with numbers kept to 22 bits and sums to 2^-24 a step, 2^-20 together at scores of
a few units; a score's own part grows with its size: its products, of signs of their own, scale sqrt(sum_d q_d^2 k_d^2) to
2^-22; and where they all have one sign, |s| itself, which the tensor cores sum in d / 16 steps, cutting the sum off below
its 24 bits (up to 2^-23 of it) at each: d / 16 2^-23 |s|. Errors
that all weights share cancel in the quotient or change a row by that part of itself; the others have signs of
their own, so that a row's error is at most about rel ||(sum_j p_j^2 v_j^2)^(1/2)|| + rel ||o||. A product that is
left out (hi x lo) would be an error of 2^-11 in the weights, a thousand times more."""
import math

import pytest

import test_gpu_paged as paged
import wcb

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TOP = {"f32": torch.finfo(torch.float32).max, "f16": torch.finfo(torch.float16).max, "bf16": torch.finfo(torch.bfloat16).max}


def exact(s, window=0, scale=0.0):
    """Of each row and head: the output in 64 bits, the bound's 2-norm for f32 activations (above), ln of the sum, and the
    bound of that."""
    scale = scale or 1 / math.sqrt(s.d)
    rep = s.h // s.hk
    q = s.q[:, :s.h * s.d].double().cpu().view(-1, s.h, s.d)
    kt, vt = s.by_token(s.k.cpu().double()), s.by_token(s.v.cpu().double())
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros(q.shape[:2], dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
    for i, (nq, nk) in enumerate(zip(s.q_len, s.kv_len)):
        if nq == 0 or nk <= 0:
            continue
        sl = s.slots(i)
        k, v = kt[sl], vt[sl]
        pos, j = torch.arange(nk - nq, nk)[:, None], torch.arange(nk)[None]
        seen = (j <= pos) & ((j > pos - window) if window else True)
        r = slice(s.start[i], s.start[i] + nq)
        for h in range(s.h):
            kk, vv, qq = k[:, h // rep], v[:, h // rep], q[r, h]
            a = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
            l = a.logsumexp(-1)
            p = torch.where(seen, (a - l[:, None]).exp(), 0.0)
            part = (qq.square() @ kk.square().T).sqrt() * abs(scale) + s.d / 32 * a.abs()
            live = p > 2.0 ** -30 * p.amax(-1, keepdim=True)
            rel = 2.0 ** -20 + 2.0 ** -22 * torch.where(live, part, 0.0).amax(-1)
            o = p @ vv
            out[r, h], lse[r, h] = o, l
            tol[r, h] = rel * (o.norm(dim=-1) + (p.square() @ vv.square()).sqrt().norm(dim=-1)) + 1e-37
            ltol[r, h] = rel + 2.0 ** -23 * l.abs().nan_to_num(0, 0, 0)
    return out, tol, lse, ltol


def check(s, rows=None, window=0, scale=0.0, more=0.0):
    """f32 activations: the rows' 2-norm errors, and their lse."""
    out, tol, lse, ltol = exact(s, window, scale)
    tol = tol + more
    rows = [r for i, n in enumerate(s.q_len) for r in range(s.start[i], s.start[i] + n)] if rows is None else rows
    got = s.out[:, :s.h * s.d].double().cpu().view(out.shape)[rows]
    assert torch.isfinite(got).all()
    far = (got - out[rows]).norm(dim=-1) / tol[rows]
    assert far.max() <= 1, (float(far.max()), rows[int(far.amax(-1).argmax())])
    assert ((s.lse.double().cpu()[rows] - lse[rows]).abs() <= ltol[rows]).all()


def put(s, i, key, k=None, v=None):
    """Key `key` of sequence i, all its heads."""
    page, slot = int(s.table[i, key // s.page]), key % s.page
    for pool, x in ((s.k, k), (s.v, v)):
        if x is not None:
            (pool[page, :, slot] if s.by_head else pool[page, slot])[:] = x


F32 = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16")]


# many rows (the tensor cores), and few (mma.sync)
@pytest.mark.parametrize("act,cache", F32)
@pytest.mark.parametrize("heads,kv_heads,dim,q", [(8, 2, 64, [70, 3]), (8, 8, 128, [70, 3]), (4, 4, 64, [6, 3])])
@pytest.mark.parametrize("size", [1e3, 1e6, 1e9, 1e30, "largest"])
@pytest.mark.parametrize("where", ["k", "v", "kv"])
def test_large_keys_and_values_that_a_row_does_not_see(gpu, act, cache, heads, kv_heads, dim, q, size, where):
    kv, window = [140, 30], 60
    s = paged.Step(q, kv, heads, kv_heads, dim, act, cache, 16, seed=50)
    size = TOP[cache] if size == "largest" else min(size, TOP[cache])
    first = kv[0] - q[0]  # the first new token's position; it alone sees the key that leaves the window after it
    for i, key in ((0, 139), (0, first - window + 1), (1, 29)):
        put(s, i, key, size if "k" in where else None, -size if "v" in where else None)
    s.attend(window=window)
    assert int(s.status.item()) == 0
    check(s, [*range(1, q[0] - 1), *range(q[0], q[0] + q[1] - 1)], window=window)


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("heads,kv_heads,dim,q", [(8, 2, 64, 80), (8, 8, 128, 80), (4, 4, 64, 6)])
@pytest.mark.parametrize("spread", [20, 40, 80])
def test_keys_and_values_of_many_sizes(gpu, act, cache, heads, kv_heads, dim, q, spread):
    """Every value has a size of its own between 1 and 2^spread, by its position: late rows see what early ones do not. Every
    eighth key is as much smaller, so that its score vanishes and is no less exact."""
    kv = 400
    s = paged.Step([q], [kv], heads, kv_heads, dim, act, cache, 16, seed=51)
    for j in range(kv):
        page, slot = int(s.table[0, j // 16]), j % 16
        s.v[page, slot] *= 2.0 ** (spread * j / kv)
        if j % 8 == 3:
            s.k[page, slot] *= 2.0 ** -spread
    s.attend()
    check(s)


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("heads,kv_heads,dim,q", [(8, 2, 64, 80), (8, 8, 128, 80)])
def test_large_values_without_weight(gpu, act, cache, heads, kv_heads, dim, q):
    """Seen values of 1e9 whose keys lie 70 nats below the others: no less exact for the rest."""
    s = paged.Step([q], [300], heads, kv_heads, dim, act, cache, 16, seed=52)
    base = torch.randn(dim, generator=torch.Generator().manual_seed(1)).cuda()
    base *= math.sqrt(dim) / base.norm()
    s.q[:, :heads * dim] = (s.q[:, :heads * dim].view(-1, heads, dim) * 0.3 + base).view(s.tokens, -1)
    for j in (5, 77, 78, 150, 219):
        put(s, 0, j, (base * -70 / math.sqrt(dim)).to(s.ct), 1e9)
    s.attend()
    check(s)


@pytest.mark.parametrize("act,cache", F32)
@pytest.mark.parametrize("heads,kv_heads,dim,q", [(4, 2, 64, 70), (4, 4, 128, 70), (4, 4, 64, 2)])
@pytest.mark.parametrize("gap", [13.0, 17.4, 25.0])
def test_a_key_that_takes_most_of_the_weight(gpu, act, cache, heads, kv_heads, dim, q, gap):
    """The first key stands `gap` nats above 12000 others and its value is zero, so that the others are the whole output."""
    s = paged.Step([q], [12000], heads, kv_heads, dim, act, cache, 64, seed=53)
    base = torch.ones(dim, device="cuda")
    s.q[:, :heads * dim] = (s.q[:, :heads * dim].view(-1, heads, dim) * 0.05 + base).view(s.tokens, -1)
    put(s, 0, 0, gap / math.sqrt(dim) * 1.0, 0.0)
    s.attend()
    check(s)


@pytest.mark.parametrize("act,cache", F32)
@pytest.mark.parametrize("heads,kv_heads,dim,q", [(8, 2, 64, 80), (8, 8, 128, 80), (4, 4, 64, 6), (8, 2, 64, 1)])
@pytest.mark.parametrize("kv", [130, 900])
def test_f32_keeps_its_low_bits(gpu, act, cache, heads, kv_heads, dim, q, kv):
    s = paged.Step([q], [kv], heads, kv_heads, dim, act, cache, 16, seed=54)
    s.attend()
    check(s)
    # one head's output over all rows, not only row by row
    out, tol, _, _ = exact(s)
    err = (s.out[:q, :s.h * s.d].double().cpu().view(q, heads, dim) - out[:q]).norm()
    assert err <= 2.0 ** -19 * out[:q].norm()


@pytest.mark.parametrize("act,cache", F32)
@pytest.mark.parametrize("heads,kv_heads,dim,q", [(4, 2, 64, 80), (4, 4, 128, 80), (4, 4, 64, 6)])
@pytest.mark.parametrize("part", ["q", "k", "p", "v"])
def test_each_low_part_counts(gpu, act, cache, heads, kv_heads, dim, q, part):
    """Numbers whose low parts all have one sign: 1 + 2^-12 (2^-10 too coarse for bf16's 8 bits: left out there) rounds to 1 in
    f16 and tf32, so that a product without its low part is off by 2^-12 of itself, and nothing averages out."""
    fine = 1 + 2.0 ** -12
    if (part in "kv" and cache != "f32"):
        pytest.skip("the cache's type has no low part")
    s = paged.Step([q], [260], heads, kv_heads, dim, act, cache, 16, seed=55)
    sign = torch.where(s.q[:, :heads * dim] < 0, -1.0, 1.0)
    s.q[:, :heads * dim] = sign * (fine if part == "q" else 1.0)
    s.k.copy_(torch.where(s.k.float() < 0, -1.0, 1.0) * (fine if part == "k" else 1.0))
    s.v.copy_(fine if part == "v" else 1.0 + (torch.arange(dim, device="cuda") % 5 == 0).float())
    if part == "p":  # two kinds of keys, weights that are no f16 numbers
        s.v[..., :dim // 2] *= torch.where(s.k.float().sum(-1, keepdim=True) > 0, 1.0, -1.0)
    s.attend(scale=0.31)
    check(s, scale=0.31)


@pytest.mark.parametrize("act,cache", paged.PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 4, 128)])
@pytest.mark.parametrize("late", [[70], [130, 190], [400, 401, 520, 700, 701]])
def test_maxima_that_move_late_and_for_some_rows(gpu, act, cache, heads, kv_heads, dim, late):
    """Keys that lie far above all before them, for every third row only: those rows' weights are made again, the others' of the
    same warp are not."""
    s = paged.Step([100], [900], heads, kv_heads, dim, act, cache, 16, seed=56)
    base = torch.randn(dim, generator=torch.Generator().manual_seed(2)).cuda()
    base /= base.norm()
    q = s.q[:, :heads * dim].view(-1, heads, dim)
    q[::3] += (3 * base).to(s.at)
    for n, j in enumerate(late):
        put(s, 0, j, (base * (6 + 5 * n) * math.sqrt(dim)).to(s.ct))
    room = s.attend()
    s.check()
    first = s.out.clone()
    for _ in range(3):
        s.out.fill_(7.0)
        s.attend(room=room)
        assert torch.equal(first, s.out)


# so many sequences that most are one CTA's from the first key to the last (a part without the first key has a maximum of its own)
@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("n,heads,kv_heads,dim,q,kv", [(12, 16, 16, 64, 40, 1500), (12, 16, 16, 128, 40, 1500), (40, 16, 16, 64, 1, 600), (40, 16, 16, 128, 1, 600),
                                                       (40, 32, 16, 64, 6, 600), (40, 32, 16, 64, 14, 600)])
@pytest.mark.parametrize("gap", [14.0, 17.7, 18.5])
def test_small_weights_beside_a_large_one(gpu, act, n, heads, kv_heads, dim, q, kv, gap):
    """A first key `gap` nats above the others (17.7: 2^-25.5), with a value of zero: the others are the whole output, and the
    sum that divides it counts them. Bound: P rounds to half a step of its type, and in f16 ends at 2^-24, which is 2^-31 of the
    largest weight: half of that a key; the scores as for f32 (their products are exact in 32 bits); one rounding."""
    s = paged.Step([q] * n, [kv] * n, heads, kv_heads, dim, act, act, 64, seed=57)
    s.q[:, :heads * dim] = (s.q[:, :heads * dim].view(-1, heads, dim) * 0.05 + 1.0).view(s.tokens, -1)
    s.k *= 0.1
    s.v.copy_(1000.0 + 100.0 * s.v.float())
    for i in range(n):
        put(s, i, 0, gap / math.sqrt(dim), 0.0)
    s.attend()
    out, tol, lse, ltol = exact(s)
    e, t = paged.half_step(s.at), n * q
    got = s.out[:t, :heads * dim].double().cpu().view(t, heads, dim)
    # (the values lie between 400 and 1600, so that o is also the sum of p |v|; the largest weight is at most 1)
    bound = out[:t] * 2.02 * e + tol[:t, :, None] + (kv * 2.0 ** -32 * 1600 + 2.0 ** -25 if act == "f16" else 0)
    assert ((got - out[:t]).abs() <= bound).all(), ((got - out[:t]).abs() / bound).max()
    assert ((s.lse.double().cpu()[:t] - lse[:t]).abs() <= ltol[:t]).all()


@pytest.mark.parametrize("cache", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,heads,kv_heads,dim,q,kv", [(12, 16, 16, 64, 40, 1500), (12, 16, 16, 128, 40, 1500), (40, 16, 16, 64, 1, 600)])
@pytest.mark.parametrize("gap", [14.0, 17.7, 25.0])
def test_small_weights_beside_a_large_one_f32(gpu, cache, n, heads, kv_heads, dim, q, kv, gap):
    """The same for f32 activations. The 63 keys that share a half tile with the large one: P is two f16 numbers with the largest
    weight of 64 keys at 2^13 or more, so that a weight is off by 2^-25 / 2^13 = 2^-38 of that one at most, its values by less
    than 2 of their largest, 1600: 64 2^-37 1600 sqrt(dim) in the 2-norm. All other keys are as exact as any."""
    s = paged.Step([q] * n, [kv] * n, heads, kv_heads, dim, "f32", cache, 64, seed=58)
    s.q[:, :heads * dim] = (s.q[:, :heads * dim].view(-1, heads, dim) * 0.05 + 1.0).view(s.tokens, -1)
    s.k *= 0.1
    s.v.copy_(1000.0 + 100.0 * s.v.float())
    for i in range(n):
        put(s, i, 0, gap / math.sqrt(dim), 0.0)
    s.attend()
    check(s, more=64 * 2.0 ** -37 * 1600 * math.sqrt(dim))


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("n,q,window", [(1, 1, 63), (4, 40, 88), (1, 100, 28), (1, 3, 61), (1, 1, 1), (1, 1, 1 << 30)])
def test_the_longest_sequence_past_its_table(gpu, act, n, q, window):
    """kv_len of 2^31 - 1 with a window that begins where the table has ended (at 2^30 keys): no key is there, so zeros and
    -infinity, whatever the places' last bits."""
    s = paged.Step([q] * n, [q] * n, 8, 2, 64, act, "f16", 16, seed=59)
    s.dev[1].fill_(2 ** 31 - 1)
    s.kv = wcb.PagedKV(s.k.data_ptr(), s.v.data_ptr(), wcb.KV_F16, 1, 1 << 30, 2, 64, 0, 0, 0)
    table = torch.zeros(n, 1, dtype=torch.int32, device="cuda") - 1  # were a key looked up, it would have no page
    s.batch = wcb.PagedBatch(s.dev[0].data_ptr(), s.dev[1].data_ptr(), table.data_ptr(), n, s.tokens, q, 1, s.status.data_ptr())
    s.attend(window=window)
    assert int(s.status.item()) == wcb.PAGED_BAD_PAGE
    assert (s.out[:n * q] == 0).all() and (s.lse[:n * q] == -math.inf).all()
    assert (s.out[n * q:] == 7).all() and (s.lse[n * q:] == 7).all()


@pytest.mark.parametrize("act,cache", paged.PAIRS)
@pytest.mark.parametrize("q", [100, 2])
@pytest.mark.parametrize("far", [1e4, 1e6, 3e7, -3e7])
def test_scores_far_from_zero(gpu, act, cache, q, far):
    """Scores of one size, far from zero and all equal: plain means of the values, and every row of the same one."""
    s = paged.Step([q], [700], 8, 2, 64, act, cache, 16, seed=60)
    s.q[:, :512] = 1.0
    s.k[:] = 1.0
    s.v.copy_(torch.where(s.v.float() < 0, 1.0, 3.0))
    scale = far / 64
    s.attend(scale=scale)
    got = s.out[:q, :512].double().cpu().view(q, 8, 64)
    vt = s.by_token(s.v.double().cpu())[s.slots(0)].repeat_interleave(4, 1)
    for r in range(0, q, 7):
        want = vt[:700 - q + r + 1].mean(0)
        # equal weights: sums of 1 and 3 are exact, so the quotient's rounding (2^-22) and the output's are left
        assert ((got[r] - want).abs() <= 3 * (paged.half_step(s.at) + 2.0 ** -22)).all(), r


@pytest.mark.parametrize("cache", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,q", [(8, 2, 64, 80), (8, 8, 128, 80)])
@pytest.mark.parametrize("small", [1e-6, 1e-12, 1e-30])
def test_dimensions_of_many_sizes(gpu, cache, heads, kv_heads, dim, q, small):
    """Half of the dimensions are `small` times the others, 8 by 8: a head's numbers share what they are measured by."""
    s = paged.Step([q], [300], heads, kv_heads, dim, "f32", cache, 16, seed=61)
    thin = (torch.arange(dim, device="cuda") // 8) % 2 == 1
    for x in (s.q[:, :heads * dim].view(-1, heads, dim), s.k, s.v):
        x[..., thin] *= small
    s.attend()
    check(s)
