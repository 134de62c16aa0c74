"""Paged serving operators (wcb_paged_append_dev, wcb_paged_attention_dev,
wcb_spec_verify_dev): everything the host refuses, before any CUDA call. The
addresses below are never dereferenced."""
import ctypes as C

import pytest

import wcb

A = 1 << 20  # a 16-byte aligned address


def pool(**o):
    a = dict(k_ptr=A, v_ptr=A, dtype=wcb.KV_F16, n_pages=8, page_size=16, n_kv_heads=4, head_dim=64)
    a.update(o)
    return wcb.PagedKV(**a)


def batch(**o):
    a = dict(q_start_ptr=A, kv_len_ptr=A, page_table_ptr=A, n_seqs=2, n_tokens=6, max_q_len=4, max_pages=4)
    a.update(o)
    return wcb.PagedBatch(**a)


def append(kv=None, b=None, rope="default", **o):
    a = dict(q_ptr=A, k_ptr=A, v_ptr=A, q_out_ptr=A + 4096, dtype=wcb.KV_F32, n_heads=8, q_stride=512, k_stride=256,
             v_stride=256, q_out_stride=512)
    a.update(o)
    wcb.paged_append_dev(kv or pool(), b or batch(), wcb.Rope(64) if rope == "default" else rope, **a)


def attend(kv=None, b=None, **o):
    a = dict(q_ptr=A, out_ptr=A + 4096, dtype=wcb.KV_F32, n_heads=8, q_stride=512, out_stride=512, workspace_ptr=A,
             workspace_bytes=1 << 40)
    a.update(o)
    wcb.paged_attention_dev(kv or pool(), b or batch(), **a)


def verify(**o):
    a = dict(draft_ptr=A, draft_len_ptr=0, target_ptr=A, draft_probs_ptr=A, u_accept_ptr=A, u_sample_ptr=A, n_seqs=2,
             max_draft=3, vocab=100, tokens_ptr=A, accepted_ptr=A)
    a.update(o)
    wcb.spec_verify_dev(**a)


def refused(words, f, *args, **kw):
    with pytest.raises(wcb.WcbError) as e:
        f(*args, **kw)
    assert e.value.code == 3 and words in e.value.message, e.value.message


POOLS = [
    (dict(dtype=3), "Unsupported data type"),
    (dict(k_ptr=0), "null"),
    (dict(v_ptr=0), "null"),
    (dict(k_ptr=A + 8), "aligned"),
    (dict(head_dim=96), "head_dim"),
    (dict(head_dim=256), "head_dim"),
    (dict(n_kv_heads=0), "n_kv_heads"),
    (dict(page_size=0), "page_size"),
    (dict(n_pages=0), "n_pages"),
    (dict(n_pages=1 << 31), "n_pages"),
    (dict(page_stride=4096, token_stride=260, head_stride=64), "multiples of 16 bytes"),
    (dict(page_stride=4096, token_stride=0, head_stride=64), "stride of 0"),
    (dict(page_stride=1 << 41, token_stride=256, head_stride=64), "2^40"),
]
BATCHES = [
    (dict(n_seqs=0), "n_seqs"),
    (dict(n_seqs=65537), "n_seqs"),
    (dict(n_tokens=0), "n_tokens"),
    (dict(n_tokens=(1 << 24) + 1), "n_tokens"),
    (dict(max_q_len=0), "max_q_len"),
    (dict(max_q_len=7), "max_q_len"),
    (dict(max_pages=0), "max_pages"),
    (dict(q_start_ptr=0), "null"),
    (dict(kv_len_ptr=0), "null"),
    (dict(page_table_ptr=0), "null"),
    (dict(page_table_ptr=A + 2), "aligned"),
    (dict(status_ptr=A + 1), "aligned"),
]


@pytest.mark.parametrize("change,words", POOLS)
def test_pools_refused(change, words):
    refused(words, append, kv=pool(**change))
    refused(words, attend, kv=pool(**change))
    refused(words, wcb.paged_attention_workspace, pool(**change), batch(), 8)


@pytest.mark.parametrize("change,words", BATCHES)
def test_batches_refused(change, words):
    refused(words, append, b=batch(**change))
    refused(words, attend, b=batch(**change))
    refused(words, wcb.paged_attention_workspace, pool(), batch(**change), 8)


def test_reserved_and_struct_sizes():
    for obj, name in ((pool(), "wcb_paged_kv"), (batch(), "wcb_paged_batch")):
        obj._c.struct_size = 8
        kw = {"kv": obj} if name == "wcb_paged_kv" else {"b": obj}
        refused(name, append, **kw)
        refused(name, attend, **kw)
    b = batch()
    b._c.reserved = 1
    refused("reserved", attend, b=b)
    r = wcb.Rope(64)
    r._c.struct_size = 16
    refused("wcb_rope", append, rope=r)
    r = wcb.Rope(64)
    r._c.reserved = 1
    refused("reserved", append, rope=r)


@pytest.mark.parametrize("act,cache,ok", [(0, 0, 1), (0, 1, 1), (0, 2, 1), (1, 1, 1), (2, 2, 1), (1, 0, 0), (1, 2, 0), (2, 0, 0),
                                          (2, 1, 0), (3, 0, 0)])
def test_type_pairs(act, cache, ok):
    # the pairs that are taken get past the types, to the next thing that is wrong
    words = "16 bytes" if ok else "Unsupported data type"
    refused(words, append, kv=pool(dtype=cache), dtype=act, q_ptr=A + 4)
    refused(words, attend, kv=pool(dtype=cache), dtype=act, q_ptr=A + 4)


@pytest.mark.parametrize("change,words", [
    (dict(q_ptr=0), "without"), (dict(n_heads=0), "without"), (dict(n_heads=4097), "n_heads"), (dict(k_ptr=0), "null"),
    (dict(v_ptr=0), "null"), (dict(q_out_ptr=0), "null"), (dict(q_stride=510), "16 bytes"), (dict(q_stride=508), "shorter"),
    (dict(k_stride=252), "shorter"), (dict(v_stride=128), "shorter"), (dict(q_out_stride=256), "shorter"), (dict(k_ptr=A + 4), "16 bytes"),
    (dict(q_out_ptr=A, q_out_stride=1024), "q's stride"), (dict(q_norm_ptr=A + 4), "aligned"), (dict(k_norm_ptr=A, eps=-1.0), "eps"),
    (dict(k_norm_ptr=A, eps=float("nan")), "eps"),
])
def test_append_refuses(change, words):
    refused(words, append, **change)


def test_rope_refuses():
    for rot, theta, halves in ((8, 1e4, 0), (144, 1e4, 0), (64, 0.0, 0), (64, -1.0, 0), (64, float("inf"), 0), (64, float("nan"), 0)):
        refused("rot_dim", wcb.Rope, rot, theta, bool(halves))
    refused("rot_dim", append, rope=wcb.Rope(128))  # the heads have 64 dimensions
    with pytest.raises(ValueError):
        wcb.Rope(64, inv_freq=[1.0])
    r = wcb.Rope(64, theta=10000.0)
    assert [r._c.inv_freq[i] for i in range(32)] == pytest.approx([10000.0 ** (-2 * i / 64) for i in range(32)], rel=1e-15)
    assert wcb.Rope(32, inv_freq=[0.5] * 16)._c.inv_freq[15] == 0.5


@pytest.mark.parametrize("change,words", [
    (dict(n_heads=0), "n_heads"), (dict(n_heads=6), "n_heads"), (dict(n_heads=4 * 65), "n_heads"), (dict(q_ptr=0), "null"), (dict(out_ptr=0), "null"),
    (dict(out_ptr=A), "out must not be q"), (dict(q_stride=500), "shorter"), (dict(out_stride=514), "16 bytes"), (dict(workspace_ptr=0), "workspace"),
    (dict(workspace_ptr=A + 8), "workspace"), (dict(workspace_bytes=4096), "workspace"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(window=(1 << 30) + 1), "window"), (dict(lse_ptr=A + 2), "lse"),
])
def test_attention_refuses(change, words):
    refused(words, attend, **change)


def test_workspace_size_is_exact():
    need = wcb.paged_attention_workspace(pool(), batch(), 8)
    assert need % 16 == 0 and need > 4096
    refused("workspace", attend, workspace_bytes=need - 1)


@pytest.mark.parametrize("change,words", [
    (dict(target_ptr=0), "null"), (dict(u_sample_ptr=0), "null"), (dict(tokens_ptr=0), "null"), (dict(accepted_ptr=0), "null"), (dict(draft_ptr=0), "null"),
    (dict(u_accept_ptr=0), "null"), (dict(n_seqs=0), "n_seqs"), (dict(n_seqs=(1 << 20) + 1), "n_seqs"), (dict(max_draft=1025), "max_draft"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 20) + 1), "vocab"), (dict(target_ptr=A + 2), "aligned"), (dict(target_row_stride=99), "shorter"), (dict(draft_row_stride=99), "shorter"),
    (dict(draft_seq_stride=1 << 41), "2^40"),
])
def test_verify_refuses(change, words):
    refused(words, verify, **change)


def test_a_null_descriptor_is_refused():
    L = wcb.lib()
    p, b, n = pool(), batch(), C.c_size_t(0)
    assert L.wcb_paged_attention_workspace(None, b._at, 8, C.byref(n)) == 3
    assert L.wcb_paged_attention_workspace(p._at, None, 8, C.byref(n)) == 3
    assert L.wcb_paged_attention_workspace(p._at, b._at, 8, None) == 3
    assert L.wcb_rope_init(None, 64, 1e4, 0) == 3
