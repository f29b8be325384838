"""Weights far below a row's maximum: one position takes nearly all of the
weight and has a value of zero (an attention sink), so that what is left of the
others is the result.  Against float64, element by element, with the bound of
test_gpu_prefix_attention.py: a score is off by at most
e = (hd + 8) 2^-24 max_j sum_d |q_d k_jd| scale, which changes a weight by a
factor within 1 +- 2e, and the weighted sum by (n + 64) 2^-24 of
sum_j p_j |v_j|: a weight that had lost bits, whatever its size, is outside."""
import numpy as np
import pytest

import paged_ref as R
from synapse_amd import hip
from test_gpu_prefix_attention import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


def place(c, group, member, i):
    """page and slot of position i of a prefix (member None) or of a suffix"""
    row = c.ptable[group] if member is None else c.table[group * c.members + member]
    return row[i // c.pool.page], i % c.pool.page


def put(c, keys, group, member, i, k0, v):
    """a position's keys (k0 in their first dim) and values [kv][hd]"""
    p, s = place(c, group, member, i)
    c.pool.k[c.layer, p, :, s] = R.store(keys, c.pool.dtype)
    c.pool.k[c.layer, p, :, s, 0] = R.store(np.float32(k0), c.pool.dtype)
    c.pool.v[c.layer, p, :, s] = R.store(v, c.pool.dtype)


def compare(c):
    hd, pool = c.pool.hd, c.pool
    c.call()
    R.sync()
    got = c.bufs["out"].download((len(c.q), c.nh * hd + 4), np.float32)[:, :c.nh * hd]
    scale, worst = 1 / np.sqrt(hd), 0.0
    for r in range(len(c.q)):
        g = r // c.members
        pl, sl = int(c.plen[g]), int(c.slen[r])
        k, v = (np.concatenate([pool.rows(x, c.layer, c.ptable[g], pl),
                                pool.rows(x, c.layer, c.table[r], sl)]) for x in "kv")
        q = c.q[r, :c.nh * hd].astype(np.float64).reshape(c.nh, hd)
        want, mag, qk = R.attention(q, k, v, scale)
        tol = (2 * (hd + 8) * 2.0 ** -24 * qk * scale + (len(k) + 64) * 2.0 ** -24) * mag
        off = np.abs(got[r].reshape(c.nh, hd) - want)
        worst = max(worst, float((off / np.maximum(mag, 1e-300)).max()))
        assert (off <= tol).all(), (r, float((off / np.maximum(tol, 1e-300)).max()))
    print("largest error of sum p|v|", worst)


def sink(dtype, kv, hd, nh, groups, members, plen, slen, orders, at, page=16, seed=1):
    """scores of a few units, and `orders` binary orders above them at position `at`"""
    c = Case(seed, dtype, page, kv, hd, nh, groups, members, plen, slen)
    c.q[:, ::hd] = 4.0
    c.pool.k[..., 0] = R.store(np.zeros(c.pool.k.shape[:-1], np.float32), dtype)
    lift = np.float32(orders * np.log(2) * np.sqrt(hd) / 4)
    zero = np.zeros((kv, hd), np.float32)
    for g in range(groups):
        if at < c.plen[g]:
            put(c, zero, g, None, at, lift, zero)
        else:
            for m in range(members):
                if at - c.plen[g] < c.slen[g * members + m]:
                    put(c, zero, g, m, at - c.plen[g], lift, zero)
    c.pool.upload()
    return c


LAYOUTS = [  # kv heads, hd, heads, groups, members, prefix, suffix
    (2, 64, 4, 1, 3, 90, 23),        # one launch, four waves
    (8, 64, 16, 3, 47, 60, 21),      # a wave a sequence
    (2, 64, 4, 1, 8, 3000, 40),      # in parts, up to 16 rows
    (1, 128, 4, 1, 7, 2100, 33),     # 28 rows
    (2, 128, 8, 2, 16, 1500, 65),    # 64 rows
    (1, 80, 3, 1, 2, 150, 30),       # dims that fill no tile
    (1, 256, 4, 1, 20, 1300, 20)]    # 80 rows of 256 dims


@pytest.mark.parametrize("orders", [10, 16, 20, 24, 28, 34, 60, 100])
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_what_a_sink_leaves(layout, orders):
    print("case", layout, orders, flush=True)
    compare(sink("f16", *layout, orders, 0))


@pytest.mark.parametrize("at", [31, 32, 63, 89, 90, 112])
@pytest.mark.parametrize("orders", [20, 30])
def test_sink_in_any_place(at, orders):
    """the first and the last position of a tile, of the prefix and of the suffix"""
    compare(sink("f16", 2, 64, 4, 1, 3, 90, 23, orders, at))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("orders", [24, 60])
def test_what_a_sink_leaves_in_other_types(dtype, orders):
    for layout in LAYOUTS[:1] + LAYOUTS[3:5]:
        compare(sink(dtype, *layout, orders, 0))


@pytest.mark.parametrize("plen", [120, 2500])
@pytest.mark.parametrize("members", [2, 20])
def test_every_level_has_dims_of_its_own(plen, members):
    """weights from 1 to 2^-105 of the largest in one tile; the values of a
    level are zero but in the dims that only it has"""
    levels = [0, 8, 17, 19, 23, 35, 37, 41, 55, 71, 90, 105]
    kv, hd, nh = 1, 128, 4
    c = Case(5, "f16", 16, kv, hd, nh, 1, members, plen, 3)
    c.q[:, :] = 0
    c.q[:, ::hd][:, :nh] = 4.0
    for g, m, total in [(0, None, plen)] + [(0, m, 3) for m in range(members)]:
        for i in range(total):
            which = (i * 5) % len(levels)
            v = np.zeros((kv, hd), np.float32)
            v[:, which * 10:which * 10 + 10] = c.rng.uniform(0.5, 2, 10)
            k0 = -levels[which] * np.log(2) * np.sqrt(hd) / 4
            put(c, np.zeros((kv, hd), np.float32), g, m, i, k0, v)
    c.pool.upload()
    compare(c)


def test_rows_of_which_some_have_a_sink():
    """rows of one tile: with and without small weights, and one that sees nothing"""
    c = sink("f16", 2, 64, 4, 2, 4, [100, 0], [5, 0, 9, 1, 0, 30, 2, 0], 26, 3)
    c.q[1::3, ::64] = -4.0   # the sink is far below the rest
    c.q[2::3, ::64] = 0.0
    compare(c)


@pytest.mark.parametrize("dtype,orders", [("f16", 22), ("f16", 110), ("bf16", 90), ("f32", 110)])
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_what_a_sink_leaves_in_pages_of_whole_tiles(layout, dtype, orders):
    """(a weight's third bf16 part is 2^-16 of it, so a bf16 pool's weights keep
    f32's bits down to 2^-110)"""
    compare(sink(dtype, *layout, orders, 0, page=64))
