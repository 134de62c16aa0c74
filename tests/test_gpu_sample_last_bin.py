"""Sampling rows whose top-k ends more than 20 temperatures below the largest logit (wcb_sample_dev): the last bin of the
kernel's count holds all of those, however far they lie."""
import numpy as np
import pytest

from test_gpu_sample import KIND, run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

STEP = 2.0 ** 43  # of the weights in sums


def strict(l, kind, t, k, p, m, u):
    """Each row against what wcb.h says, weights rounded to steps of 2^-43 for the sums. The kernel's weights are within 2^-45 of
    their value and this form's, whose quotient (l - top) / t of up to 41 is rounded, within 42 * 2^-53 < 2^-47: so both
    are within 2^-44, and each rounded weight lies between the two ends of that, lo and hi, which are the same nearly everywhere. Products of sums and
    p or u are rounded in 64 bits: a part of 2^-52. What lies in doubt by that alone may be kept or not."""
    n, v = l.shape
    got, probs, status, exact, du = run(l, kind, t, k, p, m, u)
    assert status == 0
    for i in range(n):
        x = exact[i]
        some = np.isfinite(x)
        temp, pi, mi = (float(np.float32(y[i])) for y in (t, p, m))
        e = np.where(some, np.exp((np.where(some, x, 0.0) - x[some].max()) / temp), 0.0)
        e[~some] = 0.0
        lo, hi = (np.rint(e * (1 + d) * STEP).astype(np.int64) for d in (-2.0 ** -44, 2.0 ** -44))
        order = np.argsort(np.where(some, -x, np.inf), kind="stable")[:some.sum()]
        if k[i] > 0:
            order = order[:k[i]]
        must, may = np.zeros(v, bool), np.zeros(v, bool)
        must[order] = may[order] = True
        if pi < 1:
            a, b = lo[order], hi[order]
            must[order] = np.cumsum(b) - b < pi * a.sum() * (1 - 2.0 ** -52)
            may[order] = np.cumsum(a) - a < pi * b.sum() * (1 + 2.0 ** -52)
            must[order[0]] = may[order[0]] = True
        if mi > 0:
            must &= e * (1 - 2.0 ** -44) >= min(mi, 1.0)
            may &= e * (1 + 2.0 ** -44) >= min(mi, 1.0)
        kept = probs[i] > 0
        assert not (kept & ~may).any(), (i, int(kept.sum()), int(may.sum()))
        assert not (must & ~kept & (e > 2.0 ** -58)).any(), (i, int(kept.sum()), int(must.sum()))  # below 2^-59 a weight counts as none
        if k[i] > 0:
            assert kept.sum() <= k[i], i
        a, b = lo[kept].sum(), hi[kept].sum()
        want = e[kept] * STEP / b
        assert (np.abs(probs[i][kept] - want) <= want * (2.0 ** -24 + 2.0 ** -43 + (b - a) / a)).all(), i
        # the draw: the sum up to the token exceeds u times the sum, the one before it does not (u: the largest number below 1 at most)
        y = min(max(du[i], 0.0), 1 - 2.0 ** -24)
        j = got[i]
        below = np.arange(v) <= j
        assert kept[j] and hi[j] > 0, i
        assert hi[kept & below].sum() > y * a * (1 - 2.0 ** -52) and lo[kept & below].sum() - lo[j] <= y * b * (1 + 2.0 ** -52), (i, j)
    assert run(l, kind, t, k, p, m, u, probs=False)[0] == got


# normal logits of standard deviation 2.5: the k-th lies some 10 to 40 temperatures below the largest
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,v", [(1, 1000), (1, 32000), (5, 32000), (300, 4001)])
@pytest.mark.parametrize("t", [0.1, 0.2, 0.3])
@pytest.mark.parametrize("k", [50, 700, 1000, 5000])
def test_top_k_far_below_the_largest(gpu, kind, n, v, t, k):
    r = np.random.RandomState(v + k)
    l = r.randn(n, v) * 2.5
    u = r.rand(n).tolist()
    u[0] = 0.99999994  # the last of what is kept
    for p, m in ((1.0, 0.0), (0.9, 0.0), (1.0 - 2.0 ** -20, 0.0), (1.0, 1e-9), (0.999, 1e-11)):
        strict(l, kind, [t] * n, [k] * n, [p] * n, [m] * n, u)


# a few near logits, the others all the same and far (the lowest indices of them are kept), or two far levels
@pytest.mark.parametrize("v", [260, 2000, 3000, 70001])
@pytest.mark.parametrize("far", [15.0, 19.99, 21.0, 25.0, 28.0])
@pytest.mark.parametrize("near", [1, 31, 128])
def test_equal_far_logits(gpu, v, far, near):
    r = np.random.RandomState(near)
    l = np.full((6, v), -far, np.float32)
    l[:, :near] = -r.rand(6, near)
    l[:, 0] = 0.0
    l[3:, v // 2:] -= 1.0
    strict(l, "f32", [1.0] * 6, [near + 1, near + 100, v - 1] * 2, [1.0] * 6, [0.0] * 6, [0.99999994] * 6)
    strict(l, "f32", [1.0] * 6, [near + 1, near + 100, v - 1] * 2, [1.0 - 2.0 ** -22] * 6, [0.0] * 6, [0.99999994] * 6)


# what a grammar leaves: few candidates, the others -infinity; top-k ends among them, takes all of them, or more than there are
@pytest.mark.parametrize("v", [300, 32000])
@pytest.mark.parametrize("left", [2, 12, 32, 33, 200])
@pytest.mark.parametrize("p", [1.0, 0.95, 1.0 - 2.0 ** -22])
def test_masked_rows(gpu, v, left, p):
    r = np.random.RandomState(left)
    n = 6
    l = np.full((n, v), -np.inf, np.float32)
    for i in range(n):
        at = np.sort(r.choice(v, left, replace=False))
        l[i, at] = -r.rand(left) * 35
        l[i, at[r.randint(left)]] = 0.0
    for k in (1, max(1, left // 2), left - 1, left, left + 1):
        strict(l, "f32", [1.0] * n, [k] * n, [p] * n, [0.0, 0.0, 0.0, 1e-10, 1e-12, 0.5], r.rand(n).tolist())


# weights of 2e-9 to 1e-13, many of them, count for the sums too
@pytest.mark.parametrize("n,v", [(2, 100003), (300, 3001)])
@pytest.mark.parametrize("k", [0, 1 << 20, -1])
def test_far_weights_are_summed(gpu, n, v, k):
    r = np.random.RandomState(v)
    l = (-20.5 - 8 * r.rand(n, v)).astype(np.float32)
    l[:, v // 3] = 0.0
    l[:, :v // 7] = -np.inf
    finite = int(np.isfinite(l[0]).sum())
    for kk in ([finite] * n if k < 0 else [k] * n,):
        strict(l, "f32", [1.0] * n, kk, [1.0] * n, [0.0] * n, r.rand(n).tolist())
        strict(l, "f32", [1.0] * n, kk, [1.0] * n, [1e-11] * n, r.rand(n).tolist())
