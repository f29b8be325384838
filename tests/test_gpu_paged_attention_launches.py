"""Attention of new tokens in batches that take more than one launch: tens of
thousands of sequences, few of which have tokens, and a token of each with more kv
heads than a launch has room for.  Bounds as in test_gpu_paged_attention.py."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from synapse_amd import hip
from test_gpu_paged_attention import BACK, Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


class Sparse(Case):
    """news and lens: {sequence: number} of `seqs` sequences; the tables name the pool's few pages"""

    def __init__(self, seed, dtype, page, kv, hd, nh, seqs, news, lens, max_new, max_len):
        super().__init__(seed, dtype, page, kv, hd, nh, [1], [8 * page], max_new=max_new, max_len=max_len)
        self.news, self.lens = R.i32(np.zeros(seqs)), R.i32(self.rng.integers(0, max_len + 1, seqs))
        for s, n in news.items():
            self.news[s], self.lens[s] = n, lens[s]
        self.start = R.i32(np.concatenate([[0], np.cumsum(self.news)]))
        self.tokens = int(self.news.sum()) + BACK
        self.table = R.i32(self.rng.integers(0, self.pool.pages, (seqs, -(-max_len // page))))
        self.q = self.rng.standard_normal((self.tokens, nh * hd)).astype(np.float32)


# split runs whose rows are joined in two launches; runs that are not, in two; a wave each
@pytest.mark.parametrize("case", [
    ("f16", 1024, 8, 8, 128, 16731, {0: 8, 7: 1, 16383: 3, 16384: 8, 16385: 1, 16730: 7},
     {0: 170000, 7: 90, 16383: 90000, 16384: 86000, 16385: 1, 16730: 3}, 8, 170618),
    ("bf16", 1024, 8, 8, 8, 65535, {0: 2112, 1: 1, 63548: 70, 63549: 5, 65533: 1, 65534: 66},
     {0: 2500, 1: 2900, 63548: 90, 63549: 2000, 65533: 1, 65534: 2999}, 2112, 3000)], ids=str)
def test_more_than_one_launch(case):
    print("case", case, flush=True)
    c = Sparse(1, *case)
    p, need = c.params(), C.c_size_t()
    hip.check(hip.lib().syn_hip_paged_attention_workspace(C.byref(c.pool.desc), C.byref(p), C.byref(need)))
    split = need.value > 0
    assert split == (case[-1] > 3000)
    rows = p.n_seqs * p.max_new * p.n_heads
    assert rows > (1 << 24) if split else p.n_seqs * -(-p.max_new // 64) * 8 > 1 << 24
    c.call()
    R.sync()
    c.check()
    first = c.got()
    g = R.Graph(lambda s: c.call(s))  # the same, captured and replayed
    for _ in range(3):
        c.bufs["out"].upload(np.full(first.shape, 7.0, np.float32))
        R.sync()
        g.replay()
        assert (c.got() == first).all()
    g.close()


def test_more_kv_heads_than_a_launch_holds_without_starts():
    """a wave for a token and kv head: 65535 times 1025 of them, four to a workgroup"""
    print("no starts", flush=True)
    seqs, nh, hd = 65535, 1025, 8
    assert seqs * nh > 4 * (1 << 24)
    rng = np.random.default_rng(2)
    pool = R.Pool("f16", 8, 2, 1, nh, hd, rng=rng)
    lens = R.i32(np.arange(seqs) % 9)
    one = rng.standard_normal(nh * hd).astype(np.float32)
    p = hip.PagedAttention(layer=0, n_heads=nh, n_seqs=seqs, n_tokens=seqs, max_new=1, max_len=8, window=0,
                           scale=0.0, ldq=nh * hd, ldo=nh * hd, ld_table=1)
    need = C.c_size_t()
    hip.check(hip.lib().syn_hip_paged_attention_workspace(C.byref(pool.desc), C.byref(p), C.byref(need)))
    assert need.value == 0
    q = R.dev(np.tile(one, (seqs, 1)))
    out = hip.DeviceBuffer(seqs * nh * hd * 4)
    t, n = R.dev(R.i32(np.arange(seqs) & 1)), R.dev(lens)
    hip.check(hip.lib().syn_hip_paged_attention(C.byref(pool.desc), C.byref(p), q.ptr, None, n.ptr, t.ptr,
                                                out.ptr, None, 0, None))
    R.sync()
    got = out.download((seqs, nh * hd), np.float32)
    scale = 1 / np.sqrt(hd)
    for page in range(2):
        k, v = (pool.rows(x, 0, [page], 8) for x in ("k", "v"))
        for m in range(9):
            want, mag, qk = R.attention(one.astype(np.float64).reshape(nh, hd), k[:m], v[:m], scale)
            tol = (2 * (hd + 8) * 2.0 ** -24 * qk * scale + (m + 64) * 2.0 ** -24) * mag
            rows = got[(np.arange(seqs) % 9 == m) & (np.arange(seqs) % 2 == page)]
            assert len(rows) > 3000 and (rows == rows[0]).all()
            assert (np.abs(rows[0].reshape(nh, hd) - want) <= tol).all(), (page, m)
