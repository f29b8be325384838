"""States that follow the chosen beams: moved bit for bit."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from synapse_amd import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


def moved(x, parent, w):
    """x [buffers][rows][bytes]"""
    y = x.copy()
    for r, p in enumerate(parent):
        if 0 <= p < w:
            y[:, r] = x[:, r // w * w + p]
    return y


@pytest.mark.parametrize("groups,w,row,extra,buffers,shift", [
    (1, 4, 64, 0, 1, 0), (2, 8, 131072, 0, 3, 0), (3, 5, 1000, 24, 2, 0), (1, 64, 4096, 16, 2, 0),
    (2, 3, 77, 5, 4, 1), (1, 2, 1, 0, 1, 3), (4, 16, 12, 4, 5, 4), (1, 1, 256, 0, 2, 0),
    (700, 8, 48, 0, 1, 0), (1, 33, 100003, 1, 1, 0)])
def test_rows(groups, w, row, extra, buffers, shift):
    """extra: bytes between rows that stay as they are; shift: alignment of the first"""
    rng = np.random.default_rng(groups * 1000 + w)
    stride = row + extra
    x = rng.integers(0, 256, (buffers, groups * w, stride), dtype=np.uint8)
    parent = R.i32(rng.integers(0, w, groups * w))
    parent[0] = w  # outside: stays
    if groups * w > 3:
        parent[3] = -1
    raw = np.concatenate([np.full(shift, 9, np.uint8), x.reshape(-1), np.full(32, 9, np.uint8)])
    d, dp = R.dev(raw), R.dev(parent)
    f = hip.lib().syn_hip_beam_reorder_rows
    for _ in range(2):
        hip.check(f(groups, w, dp.ptr, d.ptr + shift, row, stride, buffers, groups * w * stride, None))
        want = moved(x, parent, w)
        want[:, :, row:] = x[:, :, row:]
        x = want
    R.sync()
    got = d.download(raw.shape, np.uint8)
    assert (got[:shift] == 9).all() and (got[shift + x.size:] == 9).all()
    assert np.array_equal(got[shift:shift + x.size].reshape(x.shape), x)


def pages_step(pool, parent, held, table, spare, w):
    """the definition, in place on the host copies"""
    ps, old_table, old_k, old_v = pool.page, table.copy(), pool.k.copy(), pool.v.copy()
    for r, p in enumerate(parent):
        g = r // w
        if not 0 <= p < w:
            continue
        src = g * w + p
        n = min(max(int(held[g]), 0), table.shape[1] * ps)
        full, rest = n // ps, n % ps
        table[r, :full] = old_table[src, :full]
        if src != r and rest:
            n8 = -(-rest // 8) * 8
            a, b = old_table[src, full], spare[r]
            if 0 <= a < pool.pages and 0 <= b < pool.pages:
                pool.k[:, b, :, :n8] = old_k[:, a, :, :n8]
                pool.v[:, b, :, :n8] = old_v[:, a, :, :n8]
            spare[r], table[r, full] = old_table[r, full], b


@pytest.mark.parametrize("dtype,page,kv,hd,layers,groups,w,cols,held", [
    ("f16", 16, 2, 64, 3, 1, 4, 6, [37]), ("f32", 8, 1, 8, 1, 2, 3, 5, [0, 39]),
    ("bf16", 64, 2, 80, 2, 3, 8, 3, [64, 1, 191]), ("f16", 128, 1, 256, 2, 1, 64, 2, [129]),
    ("bf16", 16, 8, 128, 4, 2, 5, 150, [2399, 15]), ("f32", 32, 3, 40, 2, 2, 2, 4, [1000, -5]),
    ("f16", 1024, 1, 16, 1, 1, 3, 1, [1001])])
def test_pages(dtype, page, kv, hd, layers, groups, w, cols, held):
    rng = np.random.default_rng(page + w)
    rows = groups * w
    n = rows * (cols + 1) + 2
    pool = R.Pool(dtype, page, n, layers, kv, hd, rng=rng)
    ids = rng.permutation(n)[:rows * (cols + 1)]
    table, spare = R.i32(ids[:rows * cols].reshape(rows, cols)), R.i32(ids[rows * cols:])
    held = R.i32(held)
    dt, dl, ds = R.dev(table), R.dev(held), R.dev(spare)
    f = hip.lib().syn_hip_beam_reorder_pages
    for step in range(3):
        parent = R.i32(rng.integers(0, w, rows))
        if step == 1 and rows > 2:
            parent[2] = w + 3
        dp = R.dev(parent)
        hip.check(f(C.byref(pool.desc), groups, w, dp.ptr, dl.ptr, dt.ptr, cols, ds.ptr, None))
        pages_step(pool, parent, held, table, spare, w)
        R.sync()
        assert np.array_equal(dt.download(table.shape, np.int32), table)
        assert np.array_equal(ds.download(spare.shape, np.int32), spare)
        k, v = pool.download()
        assert np.array_equal(k, pool.k) and np.array_equal(v, pool.v)


def test_pages_past_32_bits():
    """a pool of over 2^32 elements: the last pages"""
    page, kv, hd, w = 512, 8, 128, 3
    far = 2 * w
    pages = (1 << 32) // (page * kv * hd) + far
    step = page * kv * hd * 2
    dk, dv = hip.DeviceBuffer(pages * step), hip.DeviceBuffer(pages * step)
    near = R.Pool("f16", page, far, 1, kv, hd, rng=np.random.default_rng(9))
    first = pages - far
    for d, x in ((dk, near.pack_k(near.k)), (dv, near.pack_v(near.v))):
        hip.check(hip.lib().syn_hip_memcpy_h2d(d.ptr + first * step, hip.ptr(x), x.nbytes))
    desc = hip.KvPages(hip.KV_F16, page, pages, 1, kv, hd, dk.ptr, dv.ptr)
    table, spare = R.i32(np.arange(w)[:, None]), R.i32(w + np.arange(w))
    parent, held = R.i32([2, 0, 0]), R.i32([301])
    d = [R.dev(a) for a in (parent, held, table + first, spare + first)]
    hip.check(hip.lib().syn_hip_beam_reorder_pages(C.byref(desc), 1, w, d[0].ptr, d[1].ptr, d[2].ptr, 1,
                                                   d[3].ptr, None))
    R.sync()
    pages_step(near, parent, held, table, spare, w)
    assert np.array_equal(d[2].download(table.shape, np.int32), table + first)
    assert np.array_equal(d[3].download(spare.shape, np.int32), spare + first)
    for b, want in ((dk, near.pack_k(near.k)), (dv, near.pack_v(near.v))):
        got = np.empty_like(want)
        hip.check(hip.lib().syn_hip_memcpy_d2h(hip.ptr(got), b.ptr + first * step, got.nbytes))
        assert np.array_equal(got, want)


def test_pages_outside_the_pool():
    rng = np.random.default_rng(5)
    pool = R.Pool("f16", 16, 10, 1, 1, 16, rng=rng)
    table, spare = R.i32([[0, -1], [1, 10], [2, 3]]), R.i32([4, 5, 2147483647])
    held, parent = R.i32([20]), R.i32([1, 2, 0])
    d = [R.dev(a) for a in (parent, held, table, spare)]
    hip.check(hip.lib().syn_hip_beam_reorder_pages(C.byref(pool.desc), 1, 3, d[0].ptr, d[1].ptr, d[2].ptr,
                                                   2, d[3].ptr, None))
    R.sync()
    pages_step(pool, parent, held, table, spare, 3)
    k, v = pool.download()
    assert np.array_equal(k, pool.k) and np.array_equal(v, pool.v)
    assert np.array_equal(d[2].download((3, 2), np.int32), table)
    assert np.array_equal(d[3].download((3,), np.int32), spare)


def test_pages_replayed_with_new_parents_and_lengths():
    rng = np.random.default_rng(6)
    w, cols = 4, 5
    pool = R.Pool("bf16", 8, w * (cols + 1), 2, 2, 16, rng=rng)
    ids = rng.permutation(w * (cols + 1))
    table, spare = R.i32(ids[:w * cols].reshape(w, cols)), R.i32(ids[w * cols:])
    parent, held = R.i32([0, 0, 1, 2]), R.i32([0])
    dp, dl, dt, ds = (R.dev(a) for a in (parent, held, table, spare))
    g = R.Graph(lambda s: hip.check(hip.lib().syn_hip_beam_reorder_pages(
        C.byref(pool.desc), 1, w, dp.ptr, dl.ptr, dt.ptr, cols, ds.ptr, s)))
    for n in range(1, 33):
        parent, held = R.i32(rng.integers(0, w, w)), R.i32([n])
        dp.upload(parent)
        dl.upload(held)
        g.replay()
        pages_step(pool, parent, held, table, spare, w)
    g.close()
    k, v = pool.download()
    assert np.array_equal(k, pool.k) and np.array_equal(v, pool.v)
    assert np.array_equal(dt.download(table.shape, np.int32), table)
    # what is to be written stays apart: every column not full yet, and the spares
    own = list(table[:, 32 // 8:].reshape(-1)) + list(spare)
    assert len(set(own)) == len(own)
