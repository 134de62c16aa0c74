"""Trees of drafted tokens and sampling (wcb_paged_tree_append_dev, wcb_paged_tree_attention_dev, wcb_tree_accept_dev,
wcb_paged_keep_dev, wcb_sample_dev): everything the host refuses, before any CUDA call (the addresses below are never
dereferenced), and wcb_paged_tree_fill."""
import numpy as np
import pytest

import wcb
from test_paged_host import A, BATCHES, POOLS, batch, pool, refused


def tree(**o):
    a = dict(depth_ptr=A, mask_ptr=A, mask_words=1)
    a.update(o)
    return wcb.PagedTree(**a)


def append(kv=None, b=None, t=None, rope="default", **o):
    a = dict(q_ptr=A, k_ptr=A, v_ptr=A, q_out_ptr=A + 4096, dtype=wcb.KV_F32, n_heads=8, q_stride=512, k_stride=256, v_stride=256, q_out_stride=512)
    a.update(o)
    wcb.paged_tree_append_dev(kv or pool(), b or batch(), t or tree(), wcb.Rope(64) if rope == "default" else rope, **a)


def attend(kv=None, b=None, t=None, **o):
    a = dict(q_ptr=A, out_ptr=A + 4096, dtype=wcb.KV_F32, n_heads=8, q_stride=512, out_stride=512, workspace_ptr=A, workspace_bytes=1 << 40)
    a.update(o)
    wcb.paged_tree_attention_dev(kv or pool(), b or batch(), t or tree(), **a)


def accept(b=None, **o):
    a = dict(parent_ptr=A, token_ptr=A, sampled_ptr=A, max_path=4, path_ptr=A, tokens_ptr=A, count_ptr=A)
    a.update(o)
    wcb.tree_accept_dev(b or batch(), **a)


def keep(kvs=None, b=None, **o):
    a = dict(path_ptr=A, max_path=4, count_ptr=A)
    a.update(o)
    wcb.paged_keep_dev(wcb.PagedLayers([pool()] if kvs is None else kvs), b or batch(), **a)


def sample(settings=None, **o):
    a = dict(logits_ptr=A, dtype=wcb.KV_F32, n_rows=2, vocab=100, u_ptr=A, tokens_ptr=A)
    a.update(o)
    s = a.pop("sampling", wcb.Sampling(*(settings or (A, A, A, A))))
    wcb.sample_dev(a.pop("logits_ptr"), a.pop("dtype"), a.pop("n_rows"), a.pop("vocab"), s, a.pop("u_ptr"), a.pop("tokens_ptr"), **a)


@pytest.mark.parametrize("change,words", POOLS)
def test_pools_refused(change, words):
    refused(words, append, kv=pool(**change))
    refused(words, attend, kv=pool(**change))
    refused(words, keep, kvs=[pool(**change)])


@pytest.mark.parametrize("change,words", BATCHES)
def test_batches_refused(change, words):
    for f in (append, attend, accept, keep):
        refused(words, f, b=batch(**change))


@pytest.mark.parametrize("f,change,words", [
    (append, dict(depth_ptr=0), "null"),
    (append, dict(depth_ptr=A + 2), "aligned"),
    (attend, dict(mask_ptr=0), "null"),
    (attend, dict(mask_ptr=A + 1), "aligned"),
    (attend, dict(mask_words=0), "mask_words"),
    (attend, dict(mask_words=(1 << 19) + 1), "mask_words"),
])
def test_trees_refused(f, change, words):
    refused(words, f, t=tree(**change))


def test_tree_parts_that_a_call_does_not_use():
    # past the tree, to the next thing that is wrong
    refused("16 bytes", append, t=tree(mask_ptr=0, mask_words=0), q_ptr=A + 4)
    refused("16 bytes", attend, t=tree(depth_ptr=0), q_ptr=A + 4)
    refused("window", attend, t=tree(depth_ptr=0), window=5)


@pytest.mark.parametrize("f", [append, attend])
@pytest.mark.parametrize("change,words", [
    (dict(dtype=wcb.KV_F16), "16 bytes"), (dict(dtype=wcb.KV_BF16), "Unsupported data type"), (dict(n_heads=5000), "n_heads"), (dict(q_stride=511), "16 bytes"),
    (dict(q_stride=256), "shorter"), (dict(q_ptr=0), "null|without")])
def test_rows_refused(f, change, words):
    o = dict(change)
    if o.get("dtype") == wcb.KV_F16:
        o["q_ptr"] = A + 4
    with pytest.raises(wcb.WcbError) as e:
        f(**o)
    assert e.value.code == 3 and any(w in e.value.message for w in words.split("|")), e.value.message


def test_struct_sizes_and_reserved():
    t = tree()
    t._c.struct_size = 8
    refused("wcb_paged_tree", append, t=t)
    refused("wcb_paged_tree", attend, t=t)
    s = wcb.Sampling()
    s._c.struct_size = 8
    refused("wcb_sampling", sample, sampling=s)
    s = wcb.Sampling()
    s._c.reserved = 1
    refused("reserved", sample, sampling=s)
    wcb.check_layouts()


@pytest.mark.parametrize("change,words", [
    (dict(workspace_ptr=0), "workspace"), (dict(workspace_ptr=A + 8), "workspace"), (dict(workspace_bytes=4096), "workspace"), (dict(lse_ptr=A + 2), "lse"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(window=(1 << 30) + 1), "window"), (dict(out_ptr=A), "out must not be q"),
    (dict(n_heads=6), "n_heads"), (dict(n_heads=0), "n_heads"), (dict(n_heads=4 * 65), "n_heads")])
def test_attention_arguments_refused(change, words):
    refused(words, attend, **change)


@pytest.mark.parametrize("change,words", [
    (dict(parent_ptr=0), "null"), (dict(token_ptr=0), "null"), (dict(sampled_ptr=0), "null"), (dict(path_ptr=0), "null"), (dict(tokens_ptr=0), "null"),
    (dict(count_ptr=0), "null"), (dict(max_path=0), "max_path"), (dict(max_path=(1 << 24) + 1), "max_path"), (dict(parent_ptr=A + 2), "aligned"),
    (dict(count_ptr=A + 1), "aligned")])
def test_accept_refused(change, words):
    refused(words, accept, **change)


@pytest.mark.parametrize("change,words", [
    (dict(path_ptr=0), "null"), (dict(count_ptr=0), "null"), (dict(max_path=0), "max_path"), (dict(path_ptr=A + 2), "aligned"), (dict(kvs=[]), "n_layers"),
    (dict(kvs=[pool(), pool(page_size=32)]), "differ"), (dict(kvs=[pool(), pool(dtype=wcb.KV_BF16)]), "differ"), (dict(kvs=[pool(), pool(n_pages=9)]), "differ"),
    (dict(kvs=[pool(), pool(page_stride=8192, token_stride=256, head_stride=64)]), "differ"), (dict(kvs=[pool(), pool(k_ptr=0)]), "null")])
def test_keep_refused(change, words):
    refused(words, keep, **change)


@pytest.mark.parametrize("change,words", [
    (dict(logits_ptr=0), "null"), (dict(u_ptr=0), "null"), (dict(tokens_ptr=0), "null"), (dict(dtype=3), "Unsupported data type"), (dict(n_rows=0), "n_rows"),
    (dict(n_rows=(1 << 20) + 1), "n_rows"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 20) + 1), "vocab"), (dict(row_stride=99), "row stride"),
    (dict(probs_ptr=A + 4096, probs_stride=99), "row stride"), (dict(row_stride=1 << 41), "2^40"), (dict(probs_ptr=A), "probs must not be logits"),
    (dict(u_ptr=A + 2), "aligned"), (dict(probs_ptr=A + 4097), "aligned"), (dict(logits_ptr=A + 2), "aligned"), (dict(settings=(A + 1, 0, 0, 0)), "aligned"),
    (dict(status_ptr=A + 3), "aligned")])
def test_sample_refused(change, words):
    refused(words, sample, **change)


@pytest.mark.parametrize("n,words", [(1, 0), (2, 1), (31, 1), (33, 0), (64, 2), (65, 0), (130, 7)])
def test_tree_fill(n, words):
    r = np.random.RandomState(n)
    parent = [-1] + [int(r.randint(0, i)) for i in range(1, n)]
    depth, mask = wcb.paged_tree_fill(parent, words)
    assert mask.shape == (n, words or -(-n // 32))
    for i in range(n):
        way, at = [i], i
        while at > 0:
            at = parent[at]
            way.append(at)
        assert depth[i] == len(way) - 1
        bits = np.unpackbits(mask[i].view(np.uint8), bitorder="little")
        assert sorted(np.flatnonzero(bits).tolist()) == sorted(way)


def test_tree_fill_refused():
    refused("earlier", wcb.paged_tree_fill, [-1, 0, 2])
    refused("earlier", wcb.paged_tree_fill, [-1, -1])
    refused("mask_words", wcb.paged_tree_fill, [-1] + [0] * 32, 1)
    refused("need 1 <= n", wcb.paged_tree_fill, [])
