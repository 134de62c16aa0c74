"""Attention of trees on both sides of the sizes at which a call takes smaller row blocks, and masks with bits that name no token."""
import pytest

from test_gpu_paged import PAIRS
from test_gpu_tree import Tree

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim,q_len", [(32, 4, 64, [26]), (32, 4, 64, [27]), (32, 4, 64, [32]), (32, 4, 64, [4] * 8), (32, 4, 64, [4] * 9), (64, 8, 128, [12]),
                                                      (64, 8, 128, [13]), (64, 8, 128, [16]), (32, 32, 128, [24]), (32, 32, 128, [25]), (32, 32, 64, [25, 1]), (1, 1, 64, [1] * 130)])
def test_blocks(gpu, act, cache, heads, kv_heads, dim, q_len):
    s = Tree(q_len, [n + 35 + 11 * i for i, n in enumerate(q_len)], heads, kv_heads, dim, act, cache, 16, True, seed=90)
    s.attend()
    s.check()
    s.attend(window=20)
    s.check(window=20)


@pytest.mark.parametrize("act,cache", PAIRS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_len", [[5, 1], [90, 3]])
def test_bits_past_the_new_tokens(gpu, act, cache, dim, q_len):
    """They name nothing, whatever lies in the slots behind the sequence (NaN here)."""
    s = Tree(q_len, [n + 30 for n in q_len], 8, 2, dim, act, cache, 64, seed=91, words=4)
    mask = s.tree_dev[1]
    for i, n in enumerate(q_len):
        for j in range(n, 128):
            mask[s.start[i]:s.start[i] + n, j // 32] |= 1 << j % 32 if j % 32 < 31 else -(1 << 31)
    s.attend()
    s.check()
