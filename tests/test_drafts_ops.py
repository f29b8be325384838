"""Refusals of the operators for sampling with drafts: every check comes before
the device is touched, so these run without a GPU.  And the definitions that the
GPU tests compare with, on cases small enough to follow by hand."""
import ctypes as C

import numpy as np
import pytest

import drafts_ref as D
from synapse_amd import hip
from test_beam_ops import ARG, BAD_PAGES, FAKE, NULL, OK, SHAPE, pages


# ---------------------------------------------------------------- attention
def attention(pg=None, ptrs=None, ws=None, ws_bytes=None, **kw):
    d = dict(layer=0, n_heads=4, n_seqs=3, n_tokens=9, max_new=4, max_len=40, window=0, scale=0.0,
             ldq=256, ldo=256, ld_table=3)
    d.update(kw)
    p, pg = hip.PagedAttention(**d), pg or pages()
    need = C.c_size_t()
    st = hip.lib().syn_hip_paged_attention_workspace(C.byref(pg), C.byref(p), C.byref(need))
    a = dict(q=FAKE, start=FAKE, len=FAKE, t=FAKE, out=2 * FAKE)
    a.update(ptrs or {})
    got = hip.lib().syn_hip_paged_attention(
        C.byref(pg), C.byref(p), *[a[x] for x in ("q", "start", "len", "t", "out")],
        FAKE if ws is None else (ws or None), need.value if ws_bytes is None else ws_bytes, None)
    return st, got


@pytest.mark.parametrize("kw,want", BAD_PAGES)
def test_attention_refuses_pages(kw, want):
    assert attention(pages(**kw)) == (want, want)


@pytest.mark.parametrize("kw,want", [
    (dict(layer=2), ARG), (dict(n_heads=0), ARG), (dict(n_heads=3), ARG),
    (dict(n_heads=70000, ldq=1 << 30, ldo=1 << 30), ARG), (dict(n_seqs=65536), ARG),
    (dict(max_len=0x7fff0001, ld_table=1 << 30), ARG), (dict(n_tokens=1 << 31), ARG),
    (dict(max_new=10), ARG), (dict(n_tokens=1 << 29, max_new=1 << 29), ARG),
    (dict(ldq=255), SHAPE), (dict(ldo=255), SHAPE), (dict(ld_table=2), SHAPE),
    (dict(max_len=49), SHAPE)])
def test_attention_refuses(kw, want):
    assert attention(**kw) == (want, want)


@pytest.mark.parametrize("kw,want", [
    (dict(ptrs=dict(q=None)), NULL), (dict(ptrs=dict(len=None)), NULL), (dict(ptrs=dict(t=None)), NULL),
    (dict(ptrs=dict(out=None)), NULL), (dict(ptrs=dict(start=None)), SHAPE),
    (dict(n_seqs=0), OK), (dict(max_new=0), OK), (dict(n_tokens=0), OK),
    (dict(n_seqs=0, ptrs=dict(q=None, out=None)), OK), (dict(n_tokens=0, ptrs=dict(q=None)), OK)])
def test_attention_refuses_calls(kw, want):
    assert attention(**kw)[1] == want


def test_attention_workspace():
    # long enough to be split over its length
    kw = dict(max_len=100000, ld_table=6250)
    assert attention(ws=0, **kw)[1] == NULL
    assert attention(ws=FAKE + 8, **kw)[1] == ARG
    assert attention(ws_bytes=16, **kw)[1] == ARG
    f = hip.lib().syn_hip_paged_attention_workspace
    assert f(C.byref(pages()), C.byref(hip.PagedAttention()), None) == NULL
    assert f(C.byref(pages()), None, C.byref(C.c_size_t())) == NULL
    assert f(None, C.byref(hip.PagedAttention()), C.byref(C.c_size_t())) == NULL


# ---------------------------------------------------------------- verification
def verify(ptrs=None, ws=None, ws_bytes=None, **kw):
    d = dict(n_seqs=3, max_draft=4, pad=0, vocab=1000, ld_target=1000, target_stride=5000,
             ld_draft=1000, draft_stride=4000)
    d.update(kw)
    p, need = hip.DraftVerify(**d), C.c_size_t()
    st = hip.lib().syn_hip_draft_verify_workspace(C.byref(p), C.byref(need))
    a = dict(target=FAKE, draft=FAKE, drafted=FAKE, n=None, heat=None, u=FAKE, token=2 * FAKE,
             count=FAKE, logp=None)
    a.update(ptrs or {})
    got = hip.lib().syn_hip_draft_verify(
        C.byref(p), *[a[x] for x in ("target", "draft", "drafted", "n", "heat", "u", "token", "count",
                                     "logp")],
        FAKE if ws is None else (ws or None), need.value if ws_bytes is None else ws_bytes, None)
    return st, got


@pytest.mark.parametrize("kw,want", [
    (dict(max_draft=65), ARG), (dict(vocab=0), ARG),
    (dict(vocab=0x7ff00001, ld_target=1 << 32, ld_draft=1 << 32), ARG), (dict(n_seqs=7282), ARG),
    (dict(ld_target=999), SHAPE), (dict(ld_draft=999), SHAPE)])
def test_verify_refuses(kw, want):
    assert verify(**kw) == (want, want)


@pytest.mark.parametrize("kw,want", [
    (dict(ptrs=dict(target=None)), NULL), (dict(ptrs=dict(drafted=None)), NULL),
    (dict(ptrs=dict(u=None)), NULL), (dict(ptrs=dict(token=None)), NULL),
    (dict(ptrs=dict(count=None)), NULL), (dict(ws=0), NULL), (dict(ws=FAKE + 8), ARG),
    (dict(ws_bytes=64), ARG), (dict(ld_draft=0), SHAPE), (dict(ptrs=dict(token=FAKE)), ARG),
    (dict(n_seqs=0), OK), (dict(n_seqs=0, ptrs=dict(target=None)), OK)])
def test_verify_refuses_calls(kw, want):
    assert verify(**kw)[1] == want


def test_verify_null_structs():
    assert hip.lib().syn_hip_draft_verify(None, *[FAKE] * 10, 0, None) == NULL
    assert hip.lib().syn_hip_draft_verify_workspace(None, C.byref(C.c_size_t())) == NULL
    assert hip.lib().syn_hip_draft_verify_workspace(C.byref(hip.DraftVerify()), None) == NULL


# ---------------------------------------------------------------- page tables
def tables(**kw):
    d = dict(page_size=16, n_pages=8, n_seqs=3, ld_table=4, table=FAKE, held=FAKE, refs=FAKE)
    d.update(kw)
    return hip.KvTables(**d)


def calls(t, pg=None, ws=FAKE, ws_bytes=1 << 20, arrays=FAKE):
    """statuses of (workspace, resize, fork)"""
    lib, need = hip.lib(), C.c_size_t()
    return (lib.syn_hip_kv_tables_workspace(C.byref(t), C.byref(need)),
            lib.syn_hip_kv_resize(C.byref(t), arrays, ws, ws_bytes, None),
            lib.syn_hip_kv_fork(C.byref(pg or pages()), C.byref(t), arrays, arrays, ws, ws_bytes, None))


@pytest.mark.parametrize("kw", [dict(page_size=4), dict(page_size=24), dict(page_size=2048),
                                dict(page_size=0), dict(n_pages=0), dict(n_pages=(1 << 24) + 1),
                                dict(n_seqs=65536), dict(n_seqs=3, ld_table=1 << 30)])
def test_tables_refused(kw):
    assert calls(tables(**kw)) == (ARG, ARG, ARG)


@pytest.mark.parametrize("kw,want", [
    (dict(t=dict(table=None)), (OK, NULL, NULL)), (dict(t=dict(held=None)), (OK, NULL, NULL)),
    (dict(t=dict(refs=None)), (OK, NULL, NULL)), (dict(arrays=None), (OK, NULL, NULL)),
    (dict(ws=None), (OK, NULL, NULL)), (dict(ws=FAKE + 8), (OK, ARG, ARG)),
    (dict(ws_bytes=8), (OK, ARG, ARG)), (dict(t=dict(n_seqs=0)), (OK, OK, OK))])
def test_table_calls_refused(kw, want):
    kw = dict(kw)
    assert calls(tables(**kw.pop("t", {})), **kw) == want


@pytest.mark.parametrize("kw,want", BAD_PAGES)
def test_fork_refuses_pages(kw, want):
    t = tables(n_pages=min(kw.get("n_pages", 8) or 8, 1 << 24))
    assert hip.lib().syn_hip_kv_fork(C.byref(pages(**kw)), C.byref(t), FAKE, FAKE, FAKE, 1 << 30, None) == want


def test_fork_refuses_other_pages():
    f = lambda t: hip.lib().syn_hip_kv_fork(C.byref(pages()), C.byref(t), FAKE, FAKE, FAKE, 1 << 20, None)
    assert f(tables(n_pages=9)) == SHAPE
    assert f(tables(page_size=32)) == SHAPE
    assert hip.lib().syn_hip_kv_fork(C.byref(pages()), None, FAKE, FAKE, FAKE, 1 << 20, None) == NULL
    assert hip.lib().syn_hip_kv_resize(None, FAKE, FAKE, 1 << 20, None) == NULL
    assert hip.lib().syn_hip_kv_tables_workspace(None, C.byref(C.c_size_t())) == NULL
    assert hip.lib().syn_hip_kv_tables_workspace(C.byref(tables()), None) == NULL


FAR = 1 << 40


def compact(a=None, t=None, b=None, u=None, live=FAKE, ws=FAKE, ws_bytes=1 << 20):
    to = dict(k=FAR, v=2 * FAR, n_pages=12)
    to.update(b or {})
    ut = dict(n_pages=12, table=2 * FAKE, held=2 * FAKE, refs=2 * FAKE)
    ut.update(u or {})
    return hip.lib().syn_hip_kv_compact(C.byref(pages(**(a or {}))), C.byref(tables(**(t or {}))),
                                        C.byref(pages(**to)), C.byref(tables(**ut)), live, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,want", [
    (dict(b=dict(dtype=hip.KV_BF16)), SHAPE), (dict(b=dict(n_layers=3)), SHAPE),
    (dict(b=dict(n_kv_heads=4)), SHAPE), (dict(b=dict(head_dim=72)), SHAPE),
    (dict(b=dict(page_size=32), u=dict(page_size=32)), SHAPE), (dict(u=dict(n_pages=8)), SHAPE),
    (dict(t=dict(n_pages=9)), SHAPE), (dict(u=dict(ld_table=3)), SHAPE), (dict(u=dict(n_seqs=4)), SHAPE),
    (dict(b=dict(k=FAKE)), ARG), (dict(b=dict(v=FAKE + 4096)), ARG), (dict(u=dict(table=FAKE)), ARG),
    (dict(u=dict(held=FAKE)), ARG), (dict(u=dict(refs=FAKE)), ARG), (dict(live=None), NULL),
    (dict(ws=None), NULL), (dict(ws=FAKE + 4), ARG), (dict(ws_bytes=8), ARG), (dict(b=dict(k=None)), NULL),
    (dict(t=dict(n_seqs=0), u=dict(n_seqs=0)), OK)])
def test_compact_refuses(kw, want):
    assert compact(**kw) == want


# ---------------------------------------------------------------- definitions
def test_verify_definition_keeps_the_target_distribution():
    """accepted and drawn tokens together are distributed as the target: the share of each first
    token over a grid of random numbers, drafts weighted by their probability"""
    rng = np.random.default_rng(5)
    target, draft = rng.standard_normal((2, 1, 5)).astype(np.float32) * 1.5
    p, q = D.softmax(target[0], 1.3), D.softmax(draft[0], 1.3)
    two, share, m = np.concatenate([target, target]), np.zeros(5), 400
    grid = ((np.arange(m) + 0.5) / m).astype(np.float32)
    for x in range(5):
        accept = min(1.0, p[x] / q[x])
        for u in grid:  # the draw after a rejection; acceptance itself is known
            t, n, _, _ = D.verify(two, draft, [x], 1, 1.3, [0.9999999, u], 0, 1)
            if accept < 0.9999:
                assert n == 1
                share[t[0]] += q[x] * (1 - accept) / m
        share[x] += q[x] * accept
    assert np.abs(share - p).max() < 5 / m


def test_table_definition():
    t = D.Tables(8, 6, 3, 3)
    t.resize([20, 8, 0])
    assert t.table.tolist() == [[0, 1, 2], [3, -1, -1], [-1, -1, -1]] and t.held.tolist() == [3, 1, 0]
    assert t.fork([0, 1, 0], [0, 0, 19]) == [(2, 4, 8)]
    assert t.table[2].tolist() == [0, 1, 4] and t.refs.tolist() == [2, 2, 1, 1, 1, 0]
    t.resize([9, 24, -1])
    assert t.table.tolist() == [[0, 1, -1], [3, 2, 5], [0, 1, 4]]
    t.resize([0, -1, 8])
    assert t.refs.tolist() == [1, 0, 1, 1, 0, 1]
    to = D.Tables(8, 3, 3, 3)
    assert t.compact(to)[0] == 4
    assert to.table.tolist() == [[-1, -1, -1], [2, 1, -1], [0, -1, -1]] and to.refs.tolist() == [1, 1, 1]
