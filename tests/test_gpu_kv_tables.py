"""Page tables of a paged cache against their definition: whole numbers and bits
of pages, all equal."""
import ctypes as C

import numpy as np
import pytest

import drafts_ref as D
import paged_ref as R
from synapse_amd import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


class Device:
    """D.Tables and the device's, with a workspace that must not be written behind."""

    def __init__(self, ref):
        self.ref = ref
        self.b = dict(table=R.dev(ref.table), held=R.dev(ref.held), refs=R.dev(ref.refs))
        self.desc = hip.KvTables(ref.page, ref.pages, len(ref.held), ref.table.shape[1], self.b["table"].ptr,
                                 self.b["held"].ptr, self.b["refs"].ptr)
        need = C.c_size_t()
        hip.check(hip.lib().syn_hip_kv_tables_workspace(C.byref(self.desc), C.byref(need)))
        self.need = need.value
        self.ws = R.dev(np.full(need.value + 256, 0xFF, np.uint8))

    def upload(self):
        for k, b in self.b.items():
            b.upload(getattr(self.ref, k))

    def resize(self, lens, stream=None):
        hip.check(hip.lib().syn_hip_kv_resize(C.byref(self.desc), lens.ptr, self.ws.ptr, self.need, stream))

    def fork(self, pool, parent, lens, stream=None):
        hip.check(hip.lib().syn_hip_kv_fork(C.byref(pool.desc), C.byref(self.desc), parent.ptr, lens.ptr,
                                            self.ws.ptr, self.need, stream))

    def check(self):
        for k, b in self.b.items():
            want = getattr(self.ref, k)
            got = b.download(want.shape, np.int32)
            assert (got == want).all(), (k, np.argwhere(got != want)[:5].tolist(), got[got != want][:5],
                                         want[got != want][:5])
        assert (self.ws.download((self.need + 256,), np.uint8)[self.need:] == 0xFF).all()


SHAPES = [  # page, pages, rows, columns
    (16, 2048, 16, 48), (8, 5, 3, 4), (16, 1, 1, 1), (64, 300, 7, 33), (16, 9000, 130, 65),
    (1024, 100, 9, 8), (16, 70000, 1030, 61), (8, 4096, 300, 13), (8, 4097, 2, 2000), (32, 250000, 40, 300),
    (8, 40, 4000, 2), (16, 30000, 8000, 3)]


@pytest.mark.parametrize("page,pages,rows,cols", SHAPES)
def test_resize(page, pages, rows, cols):
    """rows grow, shrink, end and stay; pools run out"""
    print("resize", page, pages, rows, cols, flush=True)
    rng = np.random.default_rng(pages)
    ref = D.Tables(page, pages, rows, cols)
    ref.refs[rng.random(pages) < 0.2] = 3  # the caller's own
    dev = Device(ref)
    for step in range(4):
        lens = rng.integers(0, cols * page + 1, rows)
        lens[rng.random(rows) < 0.2] = -1
        lens[rng.random(rows) < 0.1] = 0
        lens[rng.random(rows) < 0.05] = 2 ** 31 - 1
        lens = R.i32(lens)
        dev.resize(R.dev(lens))
        R.sync()
        ref.resize(lens)
        dev.check()


def test_counts_of_any_alignment():
    """counts that begin 4 bytes behind a 16-byte boundary"""
    rng = np.random.default_rng(5)
    for rows, cols, pages in ((9, 20, 210), (40, 500, 21001)):
        ref = D.Tables(16, pages, rows, cols)
        dev = Device(ref)
        buf = R.dev(np.zeros(pages + 1, np.int32))
        dev.desc.refs = buf.ptr + 4
        for _ in range(3):
            lens = R.i32(rng.integers(0, cols * 16, rows))
            dev.resize(R.dev(lens))
            R.sync()
            ref.resize(lens)
            assert (buf.download((pages + 1,), np.int32)[1:] == ref.refs).all()
            assert (dev.b["table"].download(ref.table.shape, np.int32) == ref.table).all()


def fill(ref, rng, most):
    ref.resize(rng.integers(0, most + 1, len(ref.held)))


FORKS = [  # dtype, page, pages, layers, kv, hd, rows, columns
    ("f32", 16, 200, 3, 2, 64, 9, 12), ("f16", 8, 60, 2, 1, 8, 6, 7), ("bf16", 64, 40, 2, 3, 40, 5, 3),
    ("f16", 1024, 9, 1, 1, 16, 4, 2), ("f32", 32, 500, 1, 1, 8, 70, 9), ("bf16", 16, 5000, 1, 1, 8, 300, 40),
    ("f16", 16, 12, 2, 2, 16, 8, 6)]  # (the last: pages run out)


def same(pool, copies):
    """the pool with the copies made, and the device's"""
    for a, b, n in copies:
        pool.k[:, b, :, :n] = pool.k[:, a, :, :n]
        pool.v[:, b, :, :n] = pool.v[:, a, :, :n]
    bits = lambda x: np.ascontiguousarray(x).view(np.uint8)
    k, v = pool.download()
    assert np.array_equal(bits(k), bits(pool.k)) and np.array_equal(bits(v), bits(pool.v))


@pytest.mark.parametrize("dtype,page,pages,layers,kv,hd,rows,cols", FORKS)
def test_fork(dtype, page, pages, layers, kv, hd, rows, cols):
    print("fork", dtype, page, pages, rows, cols, flush=True)
    rng = np.random.default_rng(rows)
    ref = D.Tables(page, pages, rows, cols)
    pool = R.Pool(dtype, page, pages, layers, kv, hd, rng=rng)
    fill(ref, rng, cols * page * 2 // 3)
    dev = Device(ref)
    for step in range(4):
        parent = np.arange(rows)
        some = rng.random(rows) < 0.5
        parent[some] = rng.integers(0, rows, some.sum())
        parent[rng.random(rows) < 0.1] = [-1, rows][step % 2]
        lens = rng.integers(-5, cols * page + 9, rows)
        lens[::3] = rng.integers(0, cols + 1, len(lens[::3])) * page  # whole pages
        parent, lens = R.i32(parent), R.i32(lens)
        dev.fork(pool, R.dev(parent), R.dev(lens))
        R.sync()
        copies = ref.fork(parent, lens)
        dev.check()
        same(pool, copies)
        cut = R.i32(np.where(rng.random(rows) < 0.3, rng.integers(0, cols * page, rows), -1))
        dev.resize(R.dev(cut))  # shared pages are counted down one by one
        R.sync()
        ref.resize(cut)
        dev.check()


def test_shared_pages_end_with_their_last_row():
    ref = D.Tables(8, 30, 4, 5)
    pool = R.Pool("f16", 8, 30, 1, 1, 8, rng=np.random.default_rng(1))
    ref.resize([37, 0, 0, 0])
    dev = Device(ref)
    parent, lens = R.i32([0, 0, 0, 0]), R.i32([0, 37, 37, 16])
    dev.fork(pool, R.dev(parent), R.dev(lens))
    R.sync()
    ref.fork(parent, lens)
    dev.check()
    assert ref.refs[:4].tolist() == [4, 4, 3, 3]
    for cut in ([0, -1, -1, -1], [-1, 0, -1, 0], [-1, -1, 0, -1]):
        dev.resize(R.dev(R.i32(cut)))
        R.sync()
        ref.resize(cut)
        dev.check()
    assert not ref.refs.any()


def test_bad_entries_counts_and_lengths():
    """entries outside the pool, a page named twice in a row, counts that are 0 already, held
    outside the row"""
    ref = D.Tables(8, 50, 5, 6)
    ref.resize([48, 30, 20, 10, 40])
    ref.table[0, 2], ref.table[0, 4], ref.table[1, 1] = -7, 50, 2 ** 31 - 1
    ref.table[2, 1] = ref.table[2, 0]
    ref.refs[ref.table[2, 0]] = 1
    ref.held[3], ref.held[4] = 9, -4
    ref.table[3, 2:] = [40, 41, 42, 43]
    pool = R.Pool("bf16", 8, 50, 2, 1, 16, rng=np.random.default_rng(2))
    dev = Device(ref)
    parent, lens = R.i32([0, 0, 2, 3, 3]), R.i32([0, 37, 0, 0, 29])
    dev.fork(pool, R.dev(parent), R.dev(lens))
    R.sync()
    copies = ref.fork(parent, lens)
    dev.check()
    same(pool, copies)
    cut = R.i32([3, 0, 0, 30, 48])
    dev.resize(R.dev(cut))
    R.sync()
    ref.resize(cut)
    dev.check()


COMPACT = [  # dtype, page, pages, layers, kv, hd, rows, columns, pages of the other pool, its columns
    ("f32", 16, 200, 3, 2, 64, 9, 12, 300, 12), ("f16", 8, 60, 2, 1, 8, 6, 7, 60, 9),
    ("bf16", 64, 40, 2, 3, 40, 5, 3, 9, 3), ("f16", 1024, 9, 1, 2, 128, 4, 2, 20, 2),
    ("f32", 8, 9000, 1, 1, 8, 400, 20, 8200, 700), ("bf16", 16, 30, 2, 2, 24, 3, 5, 1, 5),
    ("f16", 16, 5000, 2, 1, 8, 300, 15, 20000, 16)]


@pytest.mark.parametrize("dtype,page,pages,layers,kv,hd,rows,cols,to_pages,to_cols", COMPACT)
def test_compact(dtype, page, pages, layers, kv, hd, rows, cols, to_pages, to_cols):
    print("compact", dtype, page, pages, rows, cols, to_pages, flush=True)
    rng = np.random.default_rng(pages)
    ref, to = D.Tables(page, pages, rows, cols), D.Tables(page, to_pages, rows, to_cols)
    ref.refs[rng.random(pages) < 0.2] = 1
    pool = R.Pool(dtype, page, pages, layers, kv, hd, rng=rng)
    other = R.Pool(dtype, page, to_pages, layers, kv, hd, fill=3.0)
    fill(ref, rng, cols * page)
    parent = np.arange(rows)
    parent[rows // 2:] = rng.integers(0, rows // 2, rows - rows // 2) if rows > 1 else 0
    ref.fork(parent, rng.integers(0, cols * page, rows))
    if rows > 4:
        ref.table[1, 0] = -9  # an entry that names no page
    to.table[:], to.held[:], to.refs[:] = 99, 99, 99  # what was there before
    dev, into = Device(ref), Device(to)
    live = R.dev(np.full(1, -5, np.int32))
    for _ in range(2):
        hip.check(hip.lib().syn_hip_kv_compact(C.byref(pool.desc), C.byref(dev.desc), C.byref(other.desc),
                                               C.byref(into.desc), live.ptr, dev.ws.ptr, dev.need, None))
    R.sync()
    n, moves = ref.compact(to)
    assert live.download((1,), np.int32)[0] == n
    dev.check()
    into.check()
    for a, b in moves:
        other.k[:, b], other.v[:, b] = pool.k[:, a], pool.v[:, a]
    same(other, [])


def test_pools_past_32_bits():
    """pages whose bytes lie more than 2^32 behind the pool's, copied from and into"""
    layers, kv, hd, page, pages = 2, 8, 128, 64, 20500  # 128 KiB a page, 5.2 GiB a pool
    each = kv * hd * page * 2
    k, v, to_k, to_v = (hip.DeviceBuffer(n * each) for n in (layers * pages,) * 2 + (layers * 3,) * 2)
    pool = hip.KvPages(hip.KV_F16, page, pages, layers, kv, hd, k.ptr, v.ptr)
    rng = np.random.default_rng(3)
    ref, to = D.Tables(page, pages, 2, 4), D.Tables(page, 3, 2, 4)
    ref.table[0, :2], ref.held[0] = [pages - 1, pages - 3], 2
    ref.refs[:] = 1  # (all the caller's own, but for the last but one)
    ref.refs[pages - 2] = 0
    dev = Device(ref)

    def at(buf, layer, p):
        return buf.ptr + (layer * pages + p) * each

    data = {}
    for buf in (k, v):
        for layer in range(layers):
            for p in (pages - 1, pages - 2, pages - 3):
                x = rng.integers(0, 256, each, dtype=np.uint8)
                data[buf.ptr, layer, p] = x
                hip.check(hip.lib().syn_hip_memcpy_h2d(at(buf, layer, p), hip.ptr(x), each))

    def read(address):
        x = np.empty(each, np.uint8)
        hip.check(hip.lib().syn_hip_memcpy_d2h(hip.ptr(x), address, each))
        return x

    parent, lens = R.i32([0, 0]), R.i32([0, page + 24])
    d_parent, d_lens = R.dev(parent), R.dev(lens)
    hip.check(hip.lib().syn_hip_kv_fork(C.byref(pool), C.byref(dev.desc), d_parent.ptr, d_lens.ptr,
                                        dev.ws.ptr, dev.need, None))
    R.sync()
    assert ref.fork(parent, lens) == [(pages - 3, pages - 2, 24)]
    dev.check()
    for layer in range(layers):
        for buf, shape, take in ((k, (kv, hd // 8, page, 16), np.s_[:, :, :24]),
                                 (v, (kv, page // 8, hd, 16), np.s_[:, :3])):
            want = data[buf.ptr, layer, pages - 2].reshape(shape).copy()
            want[take] = data[buf.ptr, layer, pages - 3].reshape(shape)[take]
            assert (read(at(buf, layer, pages - 2)) == want.reshape(-1)).all()
            data[buf.ptr, layer, pages - 2] = want.reshape(-1)
    # the last three pages alone are live
    ref.refs[:pages - 3] = 0
    dev.upload()
    into, live = Device(to), R.dev(np.zeros(1, np.int32))
    other = hip.KvPages(hip.KV_F16, page, 3, layers, kv, hd, to_k.ptr, to_v.ptr)
    hip.check(hip.lib().syn_hip_kv_compact(C.byref(pool), C.byref(dev.desc), C.byref(other), C.byref(into.desc),
                                           live.ptr, dev.ws.ptr, dev.need, None))
    R.sync()
    assert ref.compact(to)[0] == 3 == live.download((1,), np.int32)[0]
    into.check()
    for layer in range(layers):
        for i in range(3):
            for a, b in ((k, to_k), (v, to_v)):
                got = read(b.ptr + (layer * 3 + i) * each)
                assert (got == data[a.ptr, layer, pages - 3 + i]).all()


def test_captured_and_replayed():
    """two graphs with a workspace each over tables of their own"""
    rng = np.random.default_rng(8)
    pool = R.Pool("f16", 16, 600, 2, 1, 16, rng=rng)
    sets = []
    for rows in (12, 30):
        ref = D.Tables(16, 600, rows, 11)
        fill(ref, rng, 100)
        dev = Device(ref)
        parent, lens, cut = (R.dev(np.zeros(rows, np.int32)) for _ in range(3))
        g = R.Graph(lambda s, d=dev, p=parent, l=lens, c=cut: (d.fork(pool, p, l, s), d.resize(c, s)))
        sets.append((ref, dev, parent, lens, cut, g))
    for _ in range(4):
        for ref, dev, parent, lens, cut, g in sets:
            n = len(ref.held)
            p, l = np.arange(n), R.i32(rng.integers(0, 170, n))
            p[n // 2:] = rng.integers(0, n // 2, n - n // 2)
            c = R.i32(np.where(rng.random(n) < 0.5, rng.integers(0, 170, n), -1))
            parent.upload(R.i32(p)), lens.upload(l), cut.upload(c)
            R.sync()
            g.replay()
            copies = ref.fork(p, l)
            ref.resize(c)
            dev.check()
            same(pool, copies)
    for s in sets:
        s[-1].close()
