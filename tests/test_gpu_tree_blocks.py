"""Attention of trees on both sides of the sizes at which a call takes smaller row blocks."""
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
