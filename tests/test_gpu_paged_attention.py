"""Causal attention of new tokens over a paged cache against float64.

Bound of an output element, from the operations in f32: a score's dot product
of hd terms (operands of 22 bits or more each) is off by at most
e = (hd + 8) 2^-24 max_j sum_d |q_d k_jd| scale, which changes every weight by
a factor within 1 +- 2e relative to the sum (weight and denominator), and the
weighted sum of n terms with its rescalings by (n + 64) 2^-24 of
sum_j p_j |v_j|."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from synapse_amd import hip

pytestmark = pytest.mark.gpu
BACK = 3  # rows of no sequence behind the last one


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


def causal(q, k, v, here, window, scale):
    """q [n][heads][hd], k and v [len][kv][hd] (NaN rows: left out), here [n] the rows' positions
    -> (out, sum of p|v|, max sum |q k| of a row and head [n][heads])"""
    n, heads, hd = q.shape
    j = np.arange(len(k))
    ok = ~np.isnan(k[:, 0, 0]) if len(k) else np.zeros(0, bool)
    seen = (j <= here[:, None]) & ok & ((j > here[:, None] - window) if window else True)
    k, v = np.where(ok[:, None, None], k, 0.0), np.where(ok[:, None, None], v, 0.0)
    out, mag, qk = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, heads))
    some = seen.any(1) if len(k) else np.zeros(n, bool)
    if not some.any():
        return out, mag, qk
    for h in range(heads):
        kk, vv = k[:, h // (heads // k.shape[1])], v[:, h // (heads // k.shape[1])]
        s = np.where(seen, scale * (q[:, h] @ kk.T), -np.inf)[some]
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[some, h], mag[some, h] = p @ vv, p @ np.abs(vv)
        qk[some, h] = np.where(seen, np.abs(q[:, h]) @ np.abs(kk).T, 0.0)[some].max(1)
    return out, mag, qk


class Case:
    def __init__(self, seed, dtype, page, kv, hd, nh, news, lens, window=0, max_new=None, max_len=None,
                 spread=1.0, pad=0, layers=2, scale=0.0, starts=True):
        rng = self.rng = np.random.default_rng(seed)
        self.nh, self.window, self.scale = nh, window, scale
        self.news, self.lens = R.i32(news), R.i32(lens)
        n = len(self.news)
        self.max_new = int(max(self.news.max(), 0)) if max_new is None else max_new
        self.max_len = int(max(self.lens.max(), 0)) if max_len is None else max_len
        self.start = R.i32(np.concatenate([[0], np.cumsum(self.news)])) if starts else None
        self.tokens = int(self.news.sum()) + (BACK if starts else 0)
        cols = -(-self.max_len // page) + 1
        self.pool = R.Pool(dtype, page, n * cols + 2, layers, kv, hd, rng=rng)
        self.table = R.i32(rng.permutation(n * cols + 2)[:n * cols].reshape(n, cols))
        self.q = (rng.standard_normal((self.tokens, nh * hd + pad)) * spread).astype(np.float32)
        self.layer = layers - 1
        self.bufs = None

    def params(self, **kw):
        d = dict(layer=self.layer, n_heads=self.nh, n_seqs=len(self.news), n_tokens=self.tokens,
                 max_new=self.max_new, max_len=self.max_len, window=self.window, scale=self.scale,
                 ldq=self.q.shape[1], ldo=self.nh * self.pool.hd + 4, ld_table=self.table.shape[1])
        d.update(kw)
        return hip.PagedAttention(**d)

    def call(self, stream=None, ws=None):
        p = self.params()
        if self.bufs is None:
            need = C.c_size_t()
            hip.check(hip.lib().syn_hip_paged_attention_workspace(C.byref(self.pool.desc), C.byref(p),
                                                                  C.byref(need)))
            self.need = need.value
            self.bufs = dict(q=R.dev(self.q), t=R.dev(self.table), l=R.dev(self.lens),
                             s=None if self.start is None else R.dev(self.start),
                             out=R.dev(np.full((self.tokens, p.ldo), 7.0, np.float32)),
                             ws=R.dev(np.full(need.value + 256, 0xFF, np.uint8)))
        b = self.bufs
        hip.check(hip.lib().syn_hip_paged_attention(
            C.byref(self.pool.desc), C.byref(p), b["q"].ptr, b["s"].ptr if b["s"] else None, b["l"].ptr,
            b["t"].ptr, b["out"].ptr, (ws or b["ws"]).ptr, self.need, stream), "paged_attention")

    def got(self):
        return self.bufs["out"].download((self.tokens, self.nh * self.pool.hd + 4), np.float32)

    def check(self, close=True):
        hd, pool, got = self.pool.hd, self.pool, self.got()
        assert (got[:, self.nh * hd:] == 7.0).all()
        tail = self.bufs["ws"].download((self.need + 256,), np.uint8)[self.need:]
        assert (tail == 0xFF).all()  # nothing behind the workspace
        scale = self.scale or 1 / np.sqrt(hd)
        done, worst = np.zeros(self.tokens, bool), 0.0
        for s in range(len(self.news)):
            if self.start is None:
                a, b = s * self.max_new, (s + 1) * self.max_new
            else:
                a, b = (int(np.clip(self.start[s + i], 0, self.tokens)) for i in (0, 1))
                b = min(max(a, b), a + self.max_new)
            if a >= b:
                continue
            n = int(np.clip(self.lens[s], 0, self.max_len))
            k, v = (pool.rows(x, self.layer, self.table[s], n) for x in ("k", "v"))
            q = self.q[a:b, :self.nh * hd].astype(np.float64).reshape(b - a, self.nh, hd)
            want, mag, qk = causal(q, k, v, n - (b - a) + np.arange(b - a), self.window, scale)
            e = (hd + 8) * 2.0 ** -24 * qk[..., None] * scale
            tol = (2 * e + (n + 64) * 2.0 ** -24) * mag
            off = np.abs(got[a:b, :self.nh * hd].reshape(b - a, self.nh, hd) - want)
            assert (off <= tol).all(), (s, np.argwhere(~(off <= tol))[:4].tolist(), float(off.max()))
            worst = max(worst, float(np.linalg.norm(off) / (np.linalg.norm(want) + 1e-30)))
            done[a:b] = True
        assert (got[~done] == 7.0).all()  # rows of no sequence
        if close:  # the operands are not rounded below f32: far inside the worst-case bound
            assert worst < 2e-5 * max(1.0, float(np.abs(self.q).max()) / 4), worst


SHAPES = [  # dtype, page, kv, hd, heads, new tokens, lengths, (window)
    ("f32", 16, 8, 128, 16, [5, 5, 5, 5], [213, 96, 5, 17]),
    ("f16", 16, 8, 128, 24, [1] * 8, [1, 2, 31, 32, 33, 1200, 64, 5]),
    ("bf16", 64, 8, 64, 32, [1, 4, 7, 2, 3], [3000, 64, 65, 2, 128]),
    ("f16", 64, 2, 128, 8, [9, 1, 64, 33], [513, 64, 64, 40]),
    ("f16", 8, 1, 8, 1, [1, 0, 1], [1, 7, 3]),
    ("bf16", 8, 2, 80, 2, [3, 8, 1], [33, 8, 9]),
    ("f32", 32, 2, 96, 6, [31, 2, 97], [31, 1500, 97]),
    ("f16", 128, 1, 256, 4, [5, 17], [129, 2000]),
    ("bf16", 1024, 1, 160, 3, [6, 40], [2300, 77]),
    ("f32", 8, 1, 256, 8, [4], [1300]),
    ("f16", 16, 2, 40, 14, [1, 2, 3], [50, 2, 1021]),
    ("f16", 16, 1, 64, 48, [2, 1], [333, 4000]),
    ("f32", 64, 1, 64, 33, [1, 3], [1200, 5]),
    ("bf16", 16, 4, 32, 4, [200, 1, 16, 15, 17, 33, 32], [200, 300, 16, 31, 17, 100, 64]),
    ("f16", 32, 1, 128, 4, [300], [900]),
    ("f16", 64, 8, 128, 24, [130, 257], [400, 257]),
    ("f16", 16, 8, 128, 32, [8, 6, 7], [2100, 9, 900], 128),
    ("bf16", 64, 2, 64, 8, [1, 1, 1], [3000, 20, 300], 1000),
    ("f32", 16, 2, 128, 4, [70, 3], [200, 100], 33),
    ("f16", 8, 1, 64, 5, [40, 1], [500, 501], 1),
    ("bf16", 32, 2, 128, 6, [100, 1], [1700, 1700], 5000),
    ("f16", 16, 2, 256, 8, [20, 5], [1000, 200], 100),
]


@pytest.mark.parametrize("case", SHAPES, ids=str)
def test_attention(case):
    print("case", case, flush=True)
    c = Case(1, *case)
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,rep", [(64, 4), (128, 2), (128, 3), (256, 1), (72, 5)])
@pytest.mark.parametrize("new", [1, 6, 12, 24])
def test_rows_of_a_tile(dtype, hd, rep, new):
    """16, 32 and 64 rows to a workgroup, whole and not; runs that are split and that are not"""
    print("rows", dtype, hd, rep, new, flush=True)
    for lens in ([new + 3, 150], [1400, new]):
        c = Case(2, dtype, 16, 2, hd, 2 * rep, [new, new], lens)
        c.call()
        R.sync()
        c.check()


def test_without_starts_and_in_strides():
    c = Case(3, "f16", 16, 2, 64, 4, [3, 3, 3], [40, 3, 700], pad=8, starts=False)
    c.call()
    R.sync()
    c.check()
    c = Case(3, "bf16", 16, 2, 64, 4, [3, 1], [40, 700], pad=3)  # rows of no alignment
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("max_len", [40, 2500])
def test_rows_that_see_nothing(dtype, max_len):
    """lengths below the number of new tokens, zero and negative; tokens above max_new"""
    c = Case(4, dtype, 8, 2, 64, 8, [5, 5, 4, 9, 2], [3, 0, -7, 40, 1], max_len=max_len, max_new=6)
    c.call()
    R.sync()
    c.check()
    got = c.got()
    assert (got[:2, :8 * 64] == 0).all() and (got[5:14, :8 * 64] == 0).all()
    assert np.abs(got[2:5, :8 * 64]).min(1).max() > 0


def test_no_position_at_all():
    c = Case(14, "f16", 8, 2, 64, 4, [3, 1], [0, 0])
    assert c.max_len == 0
    c.call()
    R.sync()
    c.check()
    assert (c.got()[:4, :256] == 0).all()


def test_starts_outside_the_rows():
    """offsets below 0, above n_tokens or falling are cut, and their rows stay"""
    c = Case(5, "f16", 16, 1, 64, 2, [4, 3, 5], [20, 30, 40])
    c.start = R.i32([-3, 2, 1 << 30, -9])
    c.max_new = 5
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("new", [1, 5, 40])
def test_pages_outside_the_pool_and_what_lies_behind(new):
    """positions in such pages are left out; slots behind a length hold NaN"""
    c = Case(6, "f16", 16, 2, 64, 8, [new, new], [200, 1500])
    for s, n in enumerate(c.lens):
        col, slot = divmod(int(n), 16)
        c.pool.k[:, c.table[s, col], :, slot:] = np.nan
        c.pool.v[:, c.table[s, col], :, slot:] = np.nan
    c.pool.upload()
    c.table[0, 3], c.table[0, 7], c.table[1, 50] = -1, c.pool.pages, 1 << 30
    c.table[1, 60:64] = -5
    c.call()
    R.sync()
    c.check()


def test_every_page_outside_the_pool():
    c = Case(7, "bf16", 16, 1, 64, 4, [3, 2], [100, 1400])
    c.table[:] = -1
    c.call()
    R.sync()
    c.check()
    assert (c.got()[:5, :256] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_steep_scores(dtype):
    """scores over many binary orders: a running maximum that moves, weights that vanish"""
    c = Case(8, dtype, 16, 2, 64, 4, [4, 30], [600, 90], spread=40.0)
    c.call()
    R.sync()
    c.check()


def test_future_positions_do_not_count():
    """huge values at positions that only later tokens see leave the earlier rows as they are"""
    c = Case(9, "f32", 16, 1, 64, 2, [8], [100])
    c.call()
    R.sync()
    before = c.got()
    for i in range(96, 100):
        c.pool.k[:, c.table[0, i // 16], :, i % 16] = 1e30
        c.pool.v[:, c.table[0, i // 16], :, i % 16] = 1e30
    c.pool.upload()
    c.call()
    R.sync()
    after = c.got()
    assert (before[:4] == after[:4]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd,new,length", [(64, 9, 100), (128, 9, 1500), (72, 40, 90), (128, 40, 2000)])
def test_rows_that_see_what_is_not_finite(dtype, bad, hd, new, length):
    """one dim of one value (or key) of a late token: the rows before it are as they were"""
    c = Case(15, dtype, 16, 2, hd, 4, [new, 3], [length, 50])
    c.call()
    R.sync()
    before = c.got()
    at, w = length - 4, 2 * hd  # seen by the last four tokens; kv head 0's rows come first
    rows = np.r_[0:new - 4, new:len(before)]
    for which in ("v", "k"):
        x = getattr(c.pool, which)
        kept = x.copy()
        x[:, c.table[0, at // 16], 1, at % 16, 5] = R.store(np.float32(bad).reshape(1), dtype)[0]
        c.pool.upload()
        c.call()
        R.sync()
        after = c.got()
        setattr(c.pool, which, kept)
        assert np.isfinite(after[rows]).all(), which
        if which == "v":
            assert (after[rows] == before[rows]).all()
            assert (after[new - 4:new, :w] == before[new - 4:new, :w]).all()
            assert (~np.isfinite(after[new - 4:new, w + 5])).all()
        else:  # (a score of +inf in a row has the others of its wave rescaled: 2e-5 as in check())
            off = np.linalg.norm(after[rows] - before[rows])
            assert off <= 4e-5 * np.linalg.norm(before[rows])


def test_one_token_is_the_prefix_operator():
    """a token a sequence: the attention of one query with an empty prefix"""
    c = Case(10, "f16", 16, 8, 128, 16, [1] * 5, [700, 33, 1, 4000, 128])
    c.call()
    R.sync()
    got = c.got()
    p = hip.PrefixAttention(layer=1, n_heads=16, n_groups=5, group_size=1, max_prefix=0,
                            max_suffix=4000, scale=0.0, ldq=2048, ldo=2052, ld_prefix_table=1,
                            ld_table=c.table.shape[1])
    need = C.c_size_t()
    lib = hip.lib()
    hip.check(lib.syn_hip_prefix_attention_workspace(C.byref(c.pool.desc), C.byref(p), C.byref(need)))
    out, ws = R.dev(np.full((5, 2052), 7.0, np.float32)), R.dev(np.zeros(need.value + 16, np.uint8))
    b = c.bufs
    hip.check(lib.syn_hip_prefix_attention(C.byref(c.pool.desc), C.byref(p), b["q"].ptr, None, None,
                                           b["t"].ptr, b["l"].ptr, out.ptr, ws.ptr, need.value, None))
    R.sync()
    want = out.download((5, 2052), np.float32)[:, :2048]
    # both within 2e-5 of the float64 value (check() above, and that operator's own tests)
    assert np.linalg.norm(got[:5, :2048] - want) < 4e-5 * np.linalg.norm(want)


def test_captured_and_replayed():
    """two graphs with a workspace each; lengths, starts and tables change between replays"""
    a = Case(11, "f16", 16, 2, 64, 8, [5, 3, 6], [300, 1800, 6], max_new=6)
    b = Case(12, "bf16", 16, 2, 128, 4, [1, 1], [900, 1100])
    graphs = []
    for c in (a, b):
        c.call()
        R.sync()
        graphs.append(R.Graph(lambda s, c=c: c.call(s)))
    for i in range(3):
        for c, g in zip((a, b), graphs):
            n = len(c.news)
            c.lens = R.i32(np.minimum(c.max_len, c.rng.integers(1, c.max_len + 1, n)))
            c.news = R.i32(c.rng.integers(0, c.max_new + 1, n))
            c.news[0] = c.max_new
            c.start = R.i32(np.concatenate([[0], np.cumsum(c.news)]))
            c.start = np.minimum(c.start, c.tokens).astype(np.int32)
            c.table = R.i32(c.rng.permutation(c.table.reshape(-1)).reshape(c.table.shape))
            c.bufs["l"].upload(c.lens)
            c.bufs["s"].upload(c.start)
            c.bufs["t"].upload(c.table)
            c.bufs["out"].upload(np.full((c.tokens, c.nh * c.pool.hd + 4), 7.0, np.float32))
        R.sync()
        for g in graphs:
            g.replay()
        for c in (a, b):
            c.check(close=False)
            first = c.got()
            c.call()  # the same, eagerly
            R.sync()
            assert (c.got() == first).all()
    for g in graphs:
        g.close()
