"""Sampling rows whose filters end, or whose weights lie, far from the largest logit (wcb_sample_dev), against the plain 64-bit
form of test_gpu_sample.py."""
import numpy as np
import pytest

import wcb
from test_gpu_sample import check, kept_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def strict(l, kind="f32", t=None, k=None, p=None, m=None, u=None, pad=0):
    """check(), and that no other tokens are kept: in both directions wherever a probability is above 2^-43 (the step of the
    weights; what weighs less may count as none), at most top_k of them, and that a row's probabilities add up to one."""
    n, v = l.shape
    got, probs = check(l, kind, t, k, p, m, u, pad)
    exact = torch.as_tensor(l).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]).double().numpy()
    for i in range(n):
        w = kept_plain(exact[i], (t or [1.0] * n)[i], (k or [0] * n)[i], (p or [1.0] * n)[i], (m or [0.0] * n)[i])
        w /= w.sum()
        assert not ((probs[i] > 2.0 ** -43) & ~(w > 0)).any() and not ((w > 2.0 ** -43) & ~(probs[i] > 0)).any(), i
        if k and k[i] > 0:
            assert (probs[i] > 0).sum() <= k[i], i
        # each is rounded once to f32, the sum of the weights has an error of half a step of 2^-43 a token
        assert abs(probs[i].sum() - 1) <= 2.0 ** -24 + 2.0 ** -40 + v * 2.0 ** -43, (i, probs[i].sum())
        assert 0 <= got[i] < v
    return got, probs


# min-p alone where a bin is less than the rounding of the largest logit over the temperature, up to what 32 bits hold
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("v", [500, 9001])
@pytest.mark.parametrize("t", [1e-3, 1e-11, 1e-12, 1e-13, 1e-20, 1e-30, 1e-45])
def test_min_p_alone_at_small_temperatures(gpu, kind, v, t):
    r = np.random.RandomState(v)
    top = np.array([20.0, 10.0, 9.7, 3.3, 0.1, -0.1, -5.0, -20.0, 1e4, -1e4, 12.34, 0.0])
    l = r.randn(len(top), v)
    l = (l - l.max(1, keepdims=True) + top[:, None]).astype(np.float32)
    n = len(top)
    strict(l, kind, [t] * n, None, None, ([0.05, 0.3, 1.0, 1e-6] * n)[:n], r.rand(n).tolist())
    strict(l, kind, [t] * n, [0] * n, [1.0] * n, [0.5] * n, r.rand(n).tolist())


@pytest.mark.parametrize("v", [40, 5001])
@pytest.mark.parametrize("top", [1e35, 3.2e36, 3.4e36, 1e37, 3.4e38, -1e37])
@pytest.mark.parametrize("t", [1.0, 1e-30, 1e35, 1e37])
def test_min_p_alone_at_large_logits(gpu, v, top, t):
    r = np.random.RandomState(v)
    l = r.randn(4, v).astype(np.float32)
    l[0, v // 2] = l[1, 0] = l[2, v - 1] = l[3, 7] = top
    if top < 0:
        with np.errstate(over="ignore"):
            l = np.abs(l) * np.float32(top)  # (the four set above become -infinity)
    l[3, 9] = l[3].max() * np.float32(1 - 0.3 * np.sign(top))
    strict(l, "f32", [t] * 4, None, None, [0.05, 1.0, 1e-3, 0.5], [0.1, 0.5, 0.99, 0.7])
