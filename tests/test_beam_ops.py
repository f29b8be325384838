"""Refusals of the beam decoding operators: every check comes before the
device is touched, so these run without a GPU."""
import ctypes as C

import pytest

from synapse_amd import hip

OK, NULL, ARG, SHAPE = 0, 1, 2, 4
FAKE = 1 << 20  # an aligned address that no refused call may read


def pages(**kw):
    d = dict(dtype=hip.KV_F16, page_size=16, n_pages=8, n_layers=2, n_kv_heads=2, head_dim=64,
             k=FAKE, v=FAKE)
    d.update(kw)
    return hip.KvPages(**d)


BAD_PAGES = [(dict(dtype=3), ARG), (dict(dtype=-1), ARG), (dict(page_size=4), ARG),
             (dict(page_size=24), ARG), (dict(page_size=2048), ARG), (dict(page_size=0), ARG),
             (dict(head_dim=0), ARG), (dict(head_dim=60), ARG), (dict(head_dim=264), ARG),
             (dict(n_kv_heads=0), ARG), (dict(n_pages=0), ARG), (dict(n_layers=0), ARG),
             (dict(n_pages=1 << 31), ARG),
             (dict(page_size=1024, head_dim=256, n_kv_heads=4096), ARG), (dict(k=None), NULL), (dict(v=None), NULL),
             (dict(k=FAKE + 4), ARG), (dict(v=FAKE + 8), ARG)]


# ---------------------------------------------------------------- append
def append(pg=None, n=3, ptrs=None, **kw):
    d = dict(layer=1, n_heads=4, n_seqs=3, rotary_dim=64, interleaved=0, n_positions=10, eps=1e-6,
             ldq=512, ldk=512, ldv=512, ldo=256, ld_table=2)
    d.update(kw)
    a = dict(q=FAKE, k=FAKE, v=FAKE, qn=None, kn=None, cos=FAKE, sin=FAKE, pos=FAKE, seq=None,
             index=FAKE, table=FAKE, out=2 * FAKE)
    a.update(ptrs or {})
    return hip.lib().syn_hip_kv_append(C.byref(pg or pages()), C.byref(hip.KvAppend(**d)), n,
                                       *[a[x] for x in ("q", "k", "v", "qn", "kn", "cos", "sin", "pos",
                                                        "seq", "index", "table", "out")], None)


@pytest.mark.parametrize("kw,want", BAD_PAGES)
def test_append_refuses_pages(kw, want):
    assert append(pages(**kw)) == want


@pytest.mark.parametrize("kw,want", [
    (dict(layer=2), ARG), (dict(rotary_dim=63), ARG), (dict(rotary_dim=66), ARG),
    (dict(ldq=255), SHAPE), (dict(ldo=255), SHAPE), (dict(ldk=127), SHAPE), (dict(ldv=127), SHAPE),
    (dict(n_heads=70000, ldq=1 << 30, ldo=1 << 30), ARG), (dict(n_seqs=1 << 31), ARG),
    (dict(n_positions=1 << 31), ARG), (dict(n=1 << 31), ARG), (dict(n=(1 << 28) - 15), ARG),
    (dict(ptrs=dict(k=None)), NULL), (dict(ptrs=dict(v=None)), NULL), (dict(ptrs=dict(q=None)), NULL),
    (dict(ptrs=dict(out=None)), NULL), (dict(ptrs=dict(cos=None)), NULL),
    (dict(ptrs=dict(sin=None)), NULL), (dict(ptrs=dict(pos=None)), NULL),
    (dict(ptrs=dict(index=None)), NULL), (dict(ptrs=dict(table=None)), NULL),
    (dict(ptrs=dict(out=FAKE)), ARG),  # in place with another stride
    (dict(n=0), OK), (dict(n=0, ptrs=dict(k=None)), OK)])
def test_append_refuses(kw, want):
    assert append(**kw) == want


def test_append_null_structs():
    f = hip.lib().syn_hip_kv_append
    assert f(None, C.byref(hip.KvAppend()), 1, *[FAKE] * 12, None) == NULL
    assert f(C.byref(pages()), None, 1, *[FAKE] * 12, None) == NULL


# ---------------------------------------------------------------- attention
def attention(pg=None, ptrs=None, ws=None, ws_bytes=None, **kw):
    d = dict(layer=0, n_heads=4, n_groups=2, group_size=3, max_prefix=40, max_suffix=20, scale=0.0,
             ldq=256, ldo=256, ld_prefix_table=3, ld_table=2)
    d.update(kw)
    p, pg = hip.PrefixAttention(**d), pg or pages()
    need = C.c_size_t()
    st = hip.lib().syn_hip_prefix_attention_workspace(C.byref(pg), C.byref(p), C.byref(need))
    a = dict(q=FAKE, pt=FAKE, pl=FAKE, t=FAKE, l=FAKE, out=FAKE)
    a.update(ptrs or {})
    got = hip.lib().syn_hip_prefix_attention(
        C.byref(pg), C.byref(p), *[a[x] for x in ("q", "pt", "pl", "t", "l", "out")],
        FAKE if ws is None else (ws or None), need.value if ws_bytes is None else ws_bytes, None)
    if st != OK:
        assert got == st  # the size and the call refuse the same descriptions
    return got


@pytest.mark.parametrize("kw,want", BAD_PAGES)
def test_attention_refuses_pages(kw, want):
    assert attention(pages(**kw)) == want


@pytest.mark.parametrize("kw,want", [
    (dict(layer=2), ARG), (dict(n_heads=3), ARG), (dict(n_heads=0), ARG), (dict(ldq=255), SHAPE),
    (dict(ldo=255), SHAPE), (dict(ld_prefix_table=2), SHAPE), (dict(ld_table=1), SHAPE),
    (dict(n_groups=70000, group_size=1), ARG), (dict(max_prefix=0xffffffff), ARG),
    (dict(max_suffix=0xffffffff), ARG), (dict(ptrs=dict(q=None)), NULL),
    # more threads than a launch holds: rows of the join, blocks of the attention
    (dict(n_groups=65535, group_size=1, n_heads=258, ldq=1 << 16, ldo=1 << 16), ARG),
    (dict(n_groups=1, group_size=65535, n_heads=512, ldq=1 << 16, ldo=1 << 16), ARG),
    (dict(ptrs=dict(out=None)), NULL), (dict(ptrs=dict(pt=None)), NULL),
    (dict(ptrs=dict(pl=None)), NULL), (dict(ptrs=dict(t=None)), NULL),
    (dict(ptrs=dict(l=None)), NULL), (dict(n_groups=0), OK), (dict(group_size=0), OK)])
def test_attention_refuses(kw, want):
    assert attention(**kw) == want


LONG = dict(max_prefix=4000, max_suffix=900, ld_prefix_table=250, ld_table=57)


@pytest.mark.parametrize("kw,want", [(dict(ws_bytes=64), ARG), (dict(ws=FAKE + 4), ARG),
                                     (dict(ws=0), NULL)])
def test_attention_refuses_workspaces(kw, want):
    """lengths that are split need one"""
    assert attention(**LONG, **kw) == want


def test_attention_null_structs():
    f = hip.lib().syn_hip_prefix_attention
    assert f(None, C.byref(hip.PrefixAttention()), *[FAKE] * 7, 0, None) == NULL
    assert f(C.byref(pages()), None, *[FAKE] * 7, 0, None) == NULL
    assert hip.lib().syn_hip_prefix_attention_workspace(C.byref(pages()), None, None) == NULL


# ---------------------------------------------------------------- choice
def select(ptrs=None, ws=FAKE, ws_bytes=None, **kw):
    d = dict(n_groups=2, n_beams=4, n_select=8, eos=1, pad=1, vocab=100, ld_logits=100)
    d.update(kw)
    p = hip.BeamSelect(**d)
    need = C.c_size_t()
    st = hip.lib().syn_hip_beam_select_workspace(C.byref(p), C.byref(need))
    a = dict(x=FAKE, s=FAKE, f=FAKE, p=FAKE, t=FAKE, v=FAKE, fo=FAKE)
    a.update(ptrs or {})
    got = hip.lib().syn_hip_beam_select(
        C.byref(p), *[a[x] for x in ("x", "s", "f", "p", "t", "v", "fo")], ws,
        need.value if ws_bytes is None else ws_bytes, None)
    if st != OK:
        assert got == st
    return got


@pytest.mark.parametrize("kw,want", [
    (dict(n_beams=0), ARG), (dict(n_beams=65), ARG), (dict(n_select=0), ARG),
    (dict(n_select=129), ARG), (dict(vocab=0), ARG), (dict(vocab=1, ld_logits=1), ARG),
    (dict(vocab=1 << 31, ld_logits=1 << 31), ARG), (dict(n_groups=20000), ARG),
    (dict(n_beams=64, n_select=128, vocab=1 << 30, ld_logits=1 << 30), ARG), (dict(ld_logits=99), SHAPE),
    (dict(pad=-1), ARG), (dict(pad=100), ARG), (dict(ptrs=dict(x=None)), NULL),
    (dict(ptrs=dict(s=None)), NULL), (dict(ptrs=dict(p=None)), NULL), (dict(ptrs=dict(t=None)), NULL),
    (dict(ptrs=dict(v=None)), NULL), (dict(ws=None), NULL), (dict(ws=FAKE + 4), ARG),
    (dict(ws_bytes=16), ARG), (dict(n_groups=0), OK)])
def test_select_refuses(kw, want):
    assert select(**kw) == want


def test_select_null_struct():
    assert hip.lib().syn_hip_beam_select(None, *[FAKE] * 8, 1 << 20, None) == NULL


# ---------------------------------------------------------------- reordering
@pytest.mark.parametrize("args,want", [
    ((2, 0, FAKE, FAKE, 64, 64, 1, 0), ARG), ((2, 65, FAKE, FAKE, 64, 64, 1, 0), ARG),
    ((40000, 2, FAKE, FAKE, 64, 64, 1, 0), ARG), ((2, 4, FAKE, FAKE, 64, 60, 1, 0), SHAPE),
    ((2, 4, FAKE, FAKE, 64, 64, 2, 511), SHAPE), ((2, 4, FAKE, FAKE, 64, 64, 70000, 512), ARG),
    ((2, 4, None, FAKE, 64, 64, 1, 0), NULL), ((2, 4, FAKE, None, 64, 64, 1, 0), NULL),
    ((1, 2, FAKE, FAKE, 1 << 36, 1 << 36, 1, 0), ARG), ((1, 2, FAKE, FAKE + 1, 1 << 32, 1 << 32, 1, 0), ARG),
    ((0, 4, None, None, 64, 64, 1, 0), OK), ((2, 4, None, None, 0, 64, 1, 0), OK),
    ((2, 4, None, None, 64, 64, 0, 0), OK)])
def test_reorder_rows_refuses(args, want):
    assert hip.lib().syn_hip_beam_reorder_rows(*args, None) == want


@pytest.mark.parametrize("kw,want", BAD_PAGES)
def test_reorder_pages_refuses_pages(kw, want):
    pg = pages(**kw)
    assert hip.lib().syn_hip_beam_reorder_pages(C.byref(pg), 1, 2, FAKE, FAKE, FAKE, 4, FAKE,
                                                None) == want


@pytest.mark.parametrize("args,want", [
    ((1, 0, FAKE, FAKE, FAKE, 4, FAKE), ARG), ((1, 65, FAKE, FAKE, FAKE, 4, FAKE), ARG),
    ((70000, 1, FAKE, FAKE, FAKE, 4, FAKE), ARG), ((1, 2, None, FAKE, FAKE, 4, FAKE), NULL),
    ((1, 2, FAKE, None, FAKE, 4, FAKE), NULL), ((1, 2, FAKE, FAKE, None, 4, FAKE), NULL),
    ((1, 2, FAKE, FAKE, FAKE, 4, None), NULL), ((1, 2, FAKE, FAKE, FAKE, 1 << 31, FAKE), ARG),
    ((1, 2, FAKE, FAKE, FAKE, 1 << 30, FAKE), ARG),
    ((0, 2, None, None, None, 4, None), OK)])
def test_reorder_pages_refuses(args, want):
    assert hip.lib().syn_hip_beam_reorder_pages(C.byref(pages()), *args, None) == want


def test_reorder_pages_refuses_more_layers_than_a_launch_holds():
    pg = pages(n_layers=1 << 24)
    assert hip.lib().syn_hip_beam_reorder_pages(C.byref(pg), 1, 2, FAKE, FAKE, FAKE, 4, FAKE, None) == ARG
