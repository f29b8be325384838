"""Batches whose sequences, counted as max_new tokens each, need more workgroups or
more joined rows than one launch takes: the workspace query, which runs on the host,
says whether a call is taken."""
import ctypes as C

import pytest

from synapse_amd import hip
from test_beam_ops import ARG, OK, pages


def query(pg, **kw):
    d = dict(layer=0, window=0, scale=0.0, ldq=kw["n_heads"] * pg.head_dim, ldo=kw["n_heads"] * pg.head_dim,
             ld_table=-(-kw["max_len"] // pg.page_size))
    d.update(kw)
    need = C.c_size_t()
    st = hip.lib().syn_hip_paged_attention_workspace(C.byref(pg), C.byref(hip.PagedAttention(**d)),
                                                     C.byref(need))
    return st, need.value


@pytest.mark.parametrize("hd,n_seqs,n_tokens,max_new,max_len", [
    (128, 512, 1535, 1024, 262144), (128, 512, 1535, 1024, 200000), (64, 600, 1499, 900, 131072),
    (64, 600, 1499, 900, 131000)])
def test_split_runs_of_many_sequences(hd, n_seqs, n_tokens, max_new, max_len):
    pg = pages(page_size=64, n_kv_heads=8, head_dim=hd, n_pages=1 << 16)
    assert query(pg, n_heads=32, n_seqs=n_seqs, n_tokens=n_tokens, max_new=max_new, max_len=max_len)[0] == OK


@pytest.mark.parametrize("nkv,rep,max_new", [(8, 4, 1000), (8, 1, 2112), (1, 16, 9000), (32, 8, 300)])
@pytest.mark.parametrize("max_len", [100, 3000, 1 << 20])
def test_many_sequences_of_few_tokens(nkv, rep, max_new, max_len):
    pg = pages(page_size=64, n_kv_heads=nkv, head_dim=64, n_pages=1 << 16)
    assert query(pg, n_heads=nkv * rep, n_seqs=65535, n_tokens=max_new + 65534, max_new=max_new,
                 max_len=max_len)[0] == OK


@pytest.mark.parametrize("nkv,rep,most", [
    (8, 1, (1 << 27) - 64), (1, 1, (1 << 27) - 64), (1, 8, (1 << 24) - 8), (9, 1, (1 << 26) - 64)])
def test_rows_of_one_sequence(nkv, rep, most):
    """a kv head's rows, up to a multiple of 64, times the kv heads, up to one of 8: 2^30 - 64"""
    pg = pages(page_size=64, n_kv_heads=nkv, head_dim=8, n_pages=1 << 16)
    for new, want in ((most, OK), (most + 1, ARG)):
        assert query(pg, n_heads=nkv * rep, n_seqs=1, n_tokens=new, max_new=new, max_len=4096)[0] == want
