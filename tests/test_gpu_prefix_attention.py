"""Attention over a shared prefix and a suffix of one's own against float64.

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


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


class Case:
    def __init__(self, seed, dtype, page, kv, hd, nh, groups, members, plen, slen, max_prefix=None,
                 max_suffix=None, spread=1.0, pad=0, layers=2, scale=0.0):
        rng = self.rng = np.random.default_rng(seed)
        self.nh, self.groups, self.members, self.scale = nh, groups, members, scale
        rows = groups * members
        self.plen = R.i32(np.broadcast_to(plen, groups))
        self.slen = R.i32(np.broadcast_to(slen, rows))
        self.max_prefix = int(max(self.plen.max(), 0)) if max_prefix is None else max_prefix
        self.max_suffix = int(max(self.slen.max(), 0)) if max_suffix is None else max_suffix
        pc, sc = -(-self.max_prefix // page) + 1, -(-self.max_suffix // page) + 1
        n = groups * pc + rows * sc
        self.pool = R.Pool(dtype, page, n + 2, layers, kv, hd, rng=rng)
        ids = rng.permutation(n + 2)[:n]
        self.ptable = R.i32(ids[:groups * pc].reshape(groups, pc))
        self.table = R.i32(ids[groups * pc:].reshape(rows, sc))
        self.q = (rng.standard_normal((rows, nh * hd + pad)) * spread).astype(np.float32)
        self.layer = layers - 1
        self.bufs = None

    def params(self, **kw):
        d = dict(layer=self.layer, n_heads=self.nh, n_groups=self.groups, group_size=self.members,
                 max_prefix=self.max_prefix, max_suffix=self.max_suffix, scale=self.scale,
                 ldq=self.q.shape[1], ldo=self.nh * self.pool.hd + 4,
                 ld_prefix_table=self.ptable.shape[1], ld_table=self.table.shape[1])
        d.update(kw)
        return hip.PrefixAttention(**d)

    def call(self, stream=None, ws=None):
        p = self.params()
        if self.bufs is None:
            need = C.c_size_t()
            hip.check(hip.lib().syn_hip_prefix_attention_workspace(C.byref(self.pool.desc),
                                                                   C.byref(p), C.byref(need)))
            self.need = need.value
            self.bufs = dict(q=R.dev(self.q), pt=R.dev(self.ptable), pl=R.dev(self.plen),
                             t=R.dev(self.table), l=R.dev(self.slen),
                             out=R.dev(np.full((len(self.q), p.ldo), 7.0, np.float32)),
                             ws=R.dev(np.full(need.value + 256, 0xFF, np.uint8)))
        b = self.bufs
        hip.check(hip.lib().syn_hip_prefix_attention(
            C.byref(self.pool.desc), C.byref(p), b["q"].ptr, b["pt"].ptr, b["pl"].ptr, b["t"].ptr,
            b["l"].ptr, b["out"].ptr, (ws or b["ws"]).ptr, self.need, stream), "prefix_attention")

    def check(self):
        hd, pool = self.pool.hd, self.pool
        got = self.bufs["out"].download((len(self.q), self.nh * hd + 4), np.float32)
        assert (got[:, self.nh * hd:] == 7.0).all()
        tail = self.bufs["ws"].download((self.need + 256,), np.uint8)[self.need:]
        assert (tail == 0xFF).all()  # nothing behind the workspace
        scale = self.scale or 1 / np.sqrt(hd)
        worst = 0.0
        for r in range(len(self.q)):
            g = r // self.members
            pl = int(np.clip(self.plen[g], 0, self.max_prefix))
            sl = int(np.clip(self.slen[r], 0, self.max_suffix))
            k = np.concatenate([pool.rows("k", self.layer, self.ptable[g], pl),
                                pool.rows("k", self.layer, self.table[r], sl)])
            v = np.concatenate([pool.rows("v", self.layer, self.ptable[g], pl),
                                pool.rows("v", self.layer, self.table[r], sl)])
            q = self.q[r, :self.nh * hd].astype(np.float64).reshape(self.nh, hd)
            want, mag, qk = R.attention(q, k, v, scale)
            e = (hd + 8) * 2.0 ** -24 * qk * scale
            tol = (2 * e + (len(k) + 64) * 2.0 ** -24) * mag
            off = np.abs(got[r, :self.nh * hd].reshape(self.nh, hd) - want)
            assert (off <= tol).all(), (r, float((off - tol).max()), float(off.max()))
            worst = max(worst, float(np.linalg.norm(off) / (np.linalg.norm(want) + 1e-30)))
        # the operands are not rounded below f32: far inside the worst-case bound
        assert worst < 2e-5 * max(1.0, float(np.abs(self.q).max()) / 4), worst


SHAPES = [  # dtype, page, kv, hd, heads, groups, members, prefix lengths, suffix lengths
    ("f32", 16, 8, 128, 16, 1, 4, 96, [17, 1, 0, 9]),
    ("f16", 16, 8, 128, 24, 1, 8, 1001, [1, 2, 31, 32, 33, 120, 64, 5]),
    ("bf16", 64, 8, 64, 32, 1, 5, 700, [300, 64, 65, 1, 128]),
    ("f16", 64, 2, 128, 8, 3, 16, [513, 64, 1], 40),
    ("f16", 8, 1, 8, 1, 2, 1, [0, 1], [0, 1]),
    ("bf16", 8, 2, 80, 2, 1, 3, 33, [8, 7, 9]),
    ("f32", 32, 2, 96, 6, 2, 2, [31, 97], [0, 0, 40, 3]),
    ("f16", 128, 1, 256, 4, 1, 2, 129, [127, 200]),
    ("bf16", 1024, 1, 160, 3, 2, 3, 300, 77),
    ("f32", 8, 1, 256, 8, 1, 1, 40, 70),
    ("f16", 16, 2, 40, 14, 1, 3, 50, 21),
    ("f16", 16, 1, 64, 48, 1, 2, 333, 19),
    ("f32", 64, 1, 64, 33, 1, 5, 200, 5),
    ("bf16", 16, 4, 32, 4, 7, 9, [200, 0, 16, 15, 17, 1, 32], 33),
    ("f16", 32, 1, 128, 4, 1, 64, 260, 9),
]


@pytest.mark.parametrize("case", SHAPES, ids=str)
def test_attention(case):
    print("case", case, flush=True)
    c = Case(1, *case)
    c.call()
    R.sync()
    c.check()


MANY = [  # more sequences' heads than workgroups run at once, little work in each
    ("f32", 16, 8, 128, 32, 2, 50, [18, 5], 2), ("f16", 8, 8, 64, 16, 3, 47, [300, 0, 9], 21),
    ("bf16", 32, 16, 40, 16, 1, 64, 0, 30), ("f16", 16, 8, 128, 24, 3, 46, [1650, 1, 900], 27),
    ("f32", 64, 8, 64, 32, 4, 60, [700, 300, 0, 33], 70), ("bf16", 16, 8, 128, 128, 2, 40, 1500, 1),
    ("bf16", 8, 32, 8, 32, 1, 40, 260, 5), ("f16", 64, 16, 256, 32, 1, 24, 80, 9)]


@pytest.mark.parametrize("case", MANY, ids=str)
def test_many_short_sequences(case):
    print("case", case, flush=True)
    c = Case(14, *case)
    c.slen[:] = c.rng.integers(0, case[-1] + 1, len(c.slen))
    c.slen[-1] = case[-1]
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_long_prefix_and_suffix(dtype):
    """long enough for any split"""
    c = Case(2, dtype, 64, 2, 64, 4, 1, 3, 9001, [5000, 1, 2049])
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_large_scores_and_rows_of_many_sizes(dtype):
    """one position takes nearly all of the weight; query rows from 1e-3 to 1e3"""
    c = Case(3, dtype, 16, 2, 64, 4, 1, 4, 200, 50)
    c.q *= np.float32([[1e-3], [1], [30], [1e3]])
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_places_past_the_lengths_are_not_read_into_the_result(dtype):
    """NaN and infinities behind the last position, in the page and in the rest of the pool"""
    c = Case(4, dtype, 16, 2, 64, 4, 1, 3, 37, [5, 18, 0])
    keep = np.zeros((c.pool.pages, 16), bool)
    for i in range(37):
        keep[c.ptable[0][i // 16], i % 16] = True
    for r, n in enumerate(c.slen):
        for i in range(n):
            keep[c.table[r][i // 16], i % 16] = True
    bad = R.store(np.float32([np.nan, np.inf, -np.inf, 3e38]), dtype)
    for x in (c.pool.k, c.pool.v):
        y = x.transpose(1, 3, 0, 2, 4)
        y[~keep] = bad[c.rng.integers(0, 4, y[~keep].shape)]
    c.pool.upload()
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("dtype,size", [("f16", 2.0 ** -20), ("f16", 2.0 ** -15), ("bf16", 2.0 ** -60),
                                        ("f32", 2.0 ** -60)])
def test_small_stored_values(dtype, size):
    """keys and values of f16 mostly below its normal range (2^-14)"""
    c = Case(11, dtype, 16, 2, 64, 4, 1, 5, 90, 33)
    c.pool.k, c.pool.v = (R.store((R.values(x, dtype) * size).astype(np.float32), dtype)
                          for x in (c.pool.k, c.pool.v))
    c.pool.upload()
    c.q *= np.float32(1 / size)
    c.call()
    R.sync()
    hd, pool = c.pool.hd, c.pool
    got = c.bufs["out"].download((5, 4 * hd + 4), np.float32)[:, :4 * hd].reshape(5, 4, hd)
    for r in range(5):
        k, v = (np.concatenate([pool.rows(x, c.layer, c.ptable[0], 90), pool.rows(x, c.layer, c.table[r], 33)])
                for x in "kv")
        q = c.q[r].astype(np.float64).reshape(4, hd)
        want, mag, qk = R.attention(q, k, v, 1 / np.sqrt(hd))
        tol = (2 * (hd + 8) * 2.0 ** -24 * qk / np.sqrt(hd) + (123 + 64) * 2.0 ** -24) * mag
        assert (np.abs(got[r] - want) <= tol).all()


@pytest.mark.parametrize("plen", [70, 1500])
def test_pool_past_32_bits(plen):
    """over 2^32 elements: a prefix and suffixes in the last pages (in one launch, and split)"""
    page, kv, hd, nh = 512, 8, 128, 16
    cols, rows = -(-plen // page), 3
    far = cols + rows
    pages = (1 << 32) // (page * kv * hd) + far
    step = page * kv * hd * 2
    dk, dv = hip.DeviceBuffer(pages * step), hip.DeviceBuffer(pages * step)
    near = R.Pool("f16", page, far, 1, kv, hd, rng=np.random.default_rng(12))
    for d, x in ((dk, near.pack_k(near.k)), (dv, near.pack_v(near.v))):
        hip.check(hip.lib().syn_hip_memcpy_h2d(d.ptr + (pages - far) * step, hip.ptr(x), x.nbytes))
    c = Case(13, "f16", page, kv, hd, nh, 1, rows, 1, 1)
    c.pool, c.layer = near, 0
    c.plen, c.slen = R.i32([plen]), R.i32([9, 33, 0])
    c.max_prefix, c.max_suffix = plen, 40
    c.ptable = R.i32(np.arange(cols)[None])
    c.table = R.i32(cols + np.arange(rows)[:, None])
    first = pages - far
    c.ptable += first
    c.table += first
    c.pool.desc = hip.KvPages(hip.KV_F16, page, pages, 1, kv, hd, dk.ptr, dv.ptr)
    c.call()
    R.sync()
    c.ptable -= first
    c.table -= first
    c.check()


def test_pages_outside_the_pool_and_odd_lengths():
    c = Case(5, "f16", 16, 2, 64, 4, 2, 2, [100, 40], [30, 20, 33, 7], max_prefix=80, max_suffix=32)
    c.plen[1], c.slen[1] = -3, -2147483648
    c.slen[0] = 2147483647
    c.ptable[0, 2], c.ptable[0, 4] = -1, c.pool.pages
    c.table[2, 0], c.table[3, 0] = 2147483647, -2147483648  # row 3: nothing is left
    c.call()
    R.sync()
    c.check()
    hd = c.pool.hd
    got = c.bufs["out"].download((4, c.nh * hd + 4), np.float32)
    assert (got[3, :c.nh * hd] == 0).all()


def test_no_prefix_and_no_suffix_at_all():
    c = Case(6, "f16", 16, 2, 64, 4, 2, 2, 0, [3, 0, 20, 1], max_prefix=0)
    c.call()
    R.sync()
    c.check()
    c = Case(6, "f16", 16, 2, 64, 4, 2, 2, [30, 0], 0, max_suffix=0)
    c.call()
    R.sync()
    c.check()
    c = Case(6, "bf16", 16, 2, 64, 4, 2, 2, 0, 0, max_prefix=0, max_suffix=0)
    c.call()
    R.sync()
    c.check()


def test_scale_and_equal_keys():
    """all scores equal: the mean of the values; a scale of one's own"""
    c = Case(7, "bf16", 16, 1, 64, 4, 1, 2, 100, [11, 0], scale=0.3, pad=9)
    c.pool.k[:] = c.pool.k[:1, :1, :1, :1]
    c.pool.upload()
    c.call()
    R.sync()
    c.check()


def test_repeats_bit_for_bit():
    c = Case(8, "f16", 16, 2, 128, 8, 2, 5, [700, 333], 90)
    c.call()
    R.sync()
    first = c.bufs["out"].download((10, 8 * 128 + 4), np.float32)
    for _ in range(3):
        c.call()
    R.sync()
    assert np.array_equal(first, c.bufs["out"].download(first.shape, np.float32))


def test_two_streams_and_replayed_graphs():
    """two captured calls with a workspace each, replayed in turn with new lengths"""
    a = Case(9, "f16", 16, 2, 64, 4, 1, 3, 900, 64, max_prefix=1000, max_suffix=80)
    b = Case(10, "bf16", 32, 2, 64, 4, 2, 2, 500, 10, max_prefix=600, max_suffix=20)
    for c in (a, b):
        c.call()
    R.sync()
    ga, gb = R.Graph(a.call), R.Graph(b.call)
    for step in range(3):
        for c in (a, b):
            c.plen = R.i32(c.rng.integers(0, c.max_prefix + 1, c.groups))
            c.slen = R.i32(c.rng.integers(0, c.max_suffix + 1, len(c.slen)))
            c.bufs["pl"].upload(c.plen)
            c.bufs["l"].upload(c.slen)
        assert ga.rt.hipGraphLaunch(ga.exec, ga.stream) == 0
        assert gb.rt.hipGraphLaunch(gb.exec, gb.stream) == 0
        R.sync()
        a.check()
        b.check()
    ga.close()
    gb.close()
