"""Keys and values into a paged cache against the definition in float64.

Tolerance, per element, in units of 2^-24: the sum of squares of a head norm
adds hd / 16 products a thread and 4 partial sums (relative error at most
hd / 16 + 6), its root halves that, and division, two products and the pair's
two roundings add at most 6; the rotation's error is relative to
|a c| + |b s|, so the bound is (hd / 32 + 12) of that sum.  A stored value may
be off by half a step of its type more (and 2^-25 absolute for f16
subnormals)."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from synapse_amd import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


def make(seed, dtype, page, kv, hd, nh, rd, n, seqs, inter=0, norm=False, stride=0, layers=2,
         aligned=False, scatter=False):
    """a batch: n tokens over `seqs` sequences, some padding"""
    rng = np.random.default_rng(seed)
    per = -(-n // seqs)
    cols = -(-(per + 40) // page)
    pool = R.Pool(dtype, page, seqs * cols + 3, layers, kv, hd, rng=rng)
    table = R.i32(rng.permutation(seqs * cols + 3)[:seqs * cols].reshape(seqs, cols))
    seq = R.i32(np.arange(n) // per)
    start = np.zeros(seqs, int) if aligned else rng.integers(0, 33, seqs)
    index = R.i32(start[seq] + np.arange(n) % per)
    if scatter:
        o = rng.permutation(n)
        seq, index = R.i32(seq[o]), R.i32(index[o])
    npos = 4096
    pos = R.i32(rng.integers(0, npos, n))
    ang = rng.uniform(-3, 3, (npos, max(rd // 2, 1))).astype(np.float32)
    ld = (nh + 2 * kv) * hd + stride
    return dict(rng=rng, pool=pool, table=table, seq=seq, index=index, pos=pos, cos=np.cos(ang),
                sin=np.sin(ang), x=rng.standard_normal((n, ld)).astype(np.float32), ld=ld, nh=nh,
                kv=kv, hd=hd, rd=rd, inter=inter, n=n, npos=npos, layer=layers - 1, eps=1e-5,
                qn=(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) if norm else None,
                kn=(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) if norm else None)


def call(b, use_seq=True, in_place=False, stream=None, bufs=None, n_seqs=None):
    nh, kv, hd = b["nh"], b["kv"], b["hd"]
    d = bufs if bufs is not None else {}
    if not d:
        for k in ("x", "pos", "seq", "index", "table", "cos", "sin", "qn", "kn"):
            d[k] = None if b[k] is None else R.dev(b[k])
        d["out"] = d["x"] if in_place else R.dev(np.full((b["n"], nh * hd + 3), 7.0, np.float32))
    ldo = b["ld"] if in_place else nh * hd + 3
    p = hip.KvAppend(layer=b["layer"], n_heads=nh, n_seqs=n_seqs or len(b["table"]), rotary_dim=b["rd"],
                     interleaved=b["inter"], n_positions=b["npos"], eps=b["eps"], ldq=b["ld"],
                     ldk=b["ld"], ldv=b["ld"], ldo=ldo, ld_table=b["table"].shape[1])
    at = lambda k: None if d[k] is None else d[k].ptr
    x = d["x"].ptr
    hip.check(hip.lib().syn_hip_kv_append(
        C.byref(b["pool"].desc), C.byref(p), b["n"], x, x + 4 * nh * hd, x + 4 * (nh + kv) * hd,
        at("qn"), at("kn"), at("cos"), at("sin"), at("pos"), at("seq") if use_seq else None,
        at("index"), at("table"), d["out"].ptr, stream), "kv_append")
    return d, ldo


def expect(b, use_seq=True, n_seqs=None):
    """out [n][nh * hd] and its bound (NaN: untouched), pools and their bounds"""
    nh, kv, hd, pool = b["nh"], b["kv"], b["hd"], b["pool"]
    x = b["x"][:, :(nh + 2 * kv) * hd].astype(np.float64).reshape(b["n"], nh + 2 * kv, hd)
    heads = x[:, :nh + kv].copy()
    if b["qn"] is not None:
        heads /= np.sqrt((heads ** 2).mean(-1, keepdims=True) + b["eps"])
        heads[:, :nh] *= b["qn"]
        heads[:, nh:] *= b["kn"]
    inside = (b["pos"] >= 0) & (b["pos"] < b["npos"])
    p = np.where(inside, b["pos"], 0)
    cos, sin = b["cos"][p].astype(np.float64)[:, None], b["sin"][p].astype(np.float64)[:, None]
    rd = b["rd"]
    turned = R.rotate(heads, cos[..., :rd // 2], sin[..., :rd // 2], rd, b["inter"])
    mag = np.abs(heads)
    mag = R.rotate(mag, np.abs(cos[..., :rd // 2]), -np.abs(sin[..., :rd // 2]), rd, b["inter"])
    mag = np.maximum(np.abs(mag), np.abs(R.rotate(np.abs(heads), np.abs(cos[..., :rd // 2]),
                                                  np.abs(sin[..., :rd // 2]), rd, b["inter"])))
    tol = (hd / 32 + 12) * 2.0 ** -24 * mag
    k, v = R.values(pool.k, pool.dtype), R.values(pool.v, pool.dtype)
    kt, vt = np.zeros(k.shape), np.zeros(v.shape)
    step = R.HALF_STEP[pool.dtype] if pool.dtype != "f32" else 0.0
    sub = 2.0 ** -25 if pool.dtype == "f16" else 0.0
    for t in range(b["n"]):
        s = b["seq"][t] if use_seq else t
        i = b["index"][t]
        if not inside[t] or i < 0 or i >= b["table"].shape[1] * pool.page:
            continue
        if not 0 <= s < (n_seqs or len(b["table"])):
            continue
        page = b["table"][s][i // pool.page]
        if not 0 <= page < pool.pages:
            continue
        k[b["layer"], page, :, i % pool.page] = turned[t, nh:]
        kt[b["layer"], page, :, i % pool.page] = (tol[t, nh:] + step * np.abs(turned[t, nh:])) * 1.01 + sub
        v[b["layer"], page, :, i % pool.page] = x[t, nh + kv:]
        vt[b["layer"], page, :, i % pool.page] = step * np.abs(x[t, nh + kv:]) * 1.01 + sub
    q = turned[:, :nh].reshape(b["n"], nh * hd).copy()
    q[~inside] = np.nan
    return q, tol[:, :nh].reshape(b["n"], nh * hd), (k, kt), (v, vt)


def check(b, d, ldo, use_seq=True, n_seqs=None, in_place=False):
    q, qt, (k, kt), (v, vt) = expect(b, use_seq, n_seqs)
    if b["nh"]:
        got = d["out"].download((b["n"], ldo), np.float32)
        skip = np.isnan(q)
        head = got[:, :q.shape[1]]
        assert (np.abs(head - q)[~skip] <= qt[~skip]).all()
        if in_place:
            assert np.array_equal(head[skip], b["x"][:, :q.shape[1]][skip])
            assert np.array_equal(got[:, q.shape[1]:], b["x"][:, q.shape[1]:])
        else:
            assert (head[skip] == 7.0).all() and (got[:, q.shape[1]:] == 7.0).all()
    gk, gv = b["pool"].download()
    for got, want, tol in ((gk, k, kt), (gv, v, vt)):
        far = np.abs(R.values(got, b["pool"].dtype) - want) - tol
        assert not (far > 0).any(), float(far.max())


SHAPES = [  # dtype, page, kv, hd, nh, rd, n, seqs, interleaved, norm, extra stride
    ("f32", 16, 8, 128, 24, 128, 1, 1, 0, False, 0),
    ("f16", 16, 8, 128, 16, 128, 8, 8, 0, True, 0),
    ("bf16", 64, 2, 64, 8, 64, 300, 3, 0, True, 5),
    ("f16", 8, 1, 8, 1, 8, 33, 2, 0, False, 1),
    ("bf16", 128, 3, 80, 6, 32, 129, 1, 1, True, 0),
    ("f32", 32, 2, 96, 2, 96, 65, 4, 1, False, 7),
    ("f16", 1024, 1, 256, 4, 128, 700, 1, 0, True, 0),
    ("bf16", 16, 2, 40, 4, 0, 50, 5, 0, False, 0),
    ("f32", 64, 5, 256, 5, 254, 19, 2, 1, True, 2),
]


@pytest.mark.parametrize("case", SHAPES, ids=str)
def test_append(case):
    print("case", case, flush=True)
    dt, page, kv, hd, nh, rd, n, seqs, inter, norm, stride = case
    b = make(1, dt, page, kv, hd, nh, rd, n, seqs, inter, norm, stride)
    d, ldo = call(b)
    R.sync()
    check(b, d, ldo)


@pytest.mark.parametrize("aligned,scatter", [(True, False), (False, False), (False, True)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_append_orders(dtype, aligned, scatter):
    """whole groups of 8 positions, prompts that begin inside one, tokens in any order"""
    b = make(2, dtype, 16, 2, 64, 4, 64, 203, 3, 0, False, 0, aligned=aligned, scatter=scatter)
    d, ldo = call(b)
    R.sync()
    check(b, d, ldo)


def test_append_decode_without_sequence_ids_and_without_queries():
    b = make(3, "f16", 16, 2, 64, 0, 64, 9, 9)
    d, ldo = call(b, use_seq=False)
    R.sync()
    check(b, d, ldo, use_seq=False)


def test_append_in_place():
    b = make(4, "bf16", 16, 2, 64, 6, 64, 37, 2, norm=True)
    d, ldo = call(b, in_place=True)
    R.sync()
    check(b, d, ldo, in_place=True)


def test_append_padding_and_places_outside():
    b = make(5, "f16", 16, 2, 64, 2, 64, 60, 3)
    b["index"][[0, 7, 30]] = -1, -2147483648, 2147483647
    b["index"][31] = b["table"].shape[1] * 16      # one past the table
    b["pos"][[3, 9, 41]] = -1, b["npos"], 2147483647
    b["seq"][[11, 12]] = -1, 3
    b["table"][1, 0], b["table"][2, 1] = -5, b["pool"].pages
    d, ldo = call(b)
    R.sync()
    check(b, d, ldo)


def test_append_overflow_and_non_finite_values():
    b = make(6, "f16", 16, 1, 8, 1, 0, 4, 1)
    b["x"][0, 8:12] = 70000.0, -70000.0, np.inf, np.nan
    b["x"][0, 16:20] = 65519.0, 65520.0, -np.inf, np.nan
    d, ldo = call(b)
    R.sync()
    gk, gv = b["pool"].download()
    p, i = b["table"][0][b["index"][0] // 16], b["index"][0] % 16
    k, v = gk[1, p, 0, i].astype(np.float64), gv[1, p, 0, i].astype(np.float64)
    assert k[0] == np.inf and k[1] == -np.inf and k[2] == np.inf and np.isnan(k[3])
    assert v[0] == 65504.0 and v[1] == np.inf and v[2] == -np.inf and np.isnan(v[3])


def test_append_past_32_bits():
    """a pool of over 2^32 elements: the last pages"""
    page, kv, hd = 1024, 8, 256
    pages = (1 << 32) // (page * kv * hd) + 2
    nbytes = pages * page * kv * hd * 2
    k, v = hip.DeviceBuffer(nbytes), hip.DeviceBuffer(nbytes)
    desc = hip.KvPages(hip.KV_F16, page, pages, 1, kv, hd, k.ptr, v.ptr)
    rng = np.random.default_rng(7)
    n = 17
    x = rng.standard_normal((n, 2 * kv * hd)).astype(np.float32)
    index = R.i32(np.arange(n) + 1000)
    table = R.i32([[pages - 1, pages - 2]])
    z, pos = R.dev(np.zeros((1, 1), np.float32)), R.dev(np.zeros(n, np.int32))
    bx, bi, bt = R.dev(x), R.dev(index), R.dev(table)
    p = hip.KvAppend(layer=0, n_heads=0, n_seqs=1, rotary_dim=0, interleaved=0, n_positions=1, eps=0,
                     ldq=0, ldk=2 * kv * hd, ldv=2 * kv * hd, ldo=0, ld_table=2)
    seq = R.dev(np.zeros(n, np.int32))
    hip.check(hip.lib().syn_hip_kv_append(C.byref(desc), C.byref(p), n, None, bx.ptr,
                                          bx.ptr + 4 * kv * hd, None, None, z.ptr, z.ptr, pos.ptr,
                                          seq.ptr, bi.ptr, bt.ptr, None, None))
    R.sync()
    host = np.empty((2, kv, hd // 8, page, 8), np.float16)
    hostv = np.empty((2, kv, page // 8, hd, 8), np.float16)
    off = (pages - 2) * page * kv * hd * 2
    hip.check(hip.lib().syn_hip_memcpy_d2h(hip.ptr(host), k.ptr + off, host.nbytes))
    hip.check(hip.lib().syn_hip_memcpy_d2h(hip.ptr(hostv), v.ptr + off, hostv.nbytes))
    for t in range(n):
        i = int(index[t])
        pg = 1 if i < page else 0  # table column 0 is the last page of the pool
        want = x[t].astype(np.float16).reshape(2, kv, hd)
        assert np.array_equal(host[pg, :, :, i % page].reshape(kv, hd), want[0])
        assert np.array_equal(hostv[pg, :, i % page // 8, :, i % 8], want[1])


def test_append_replayed_with_new_positions():
    b = make(8, "f16", 16, 2, 64, 4, 64, 6, 6, norm=True)
    d, ldo = call(b)  # buffers
    R.sync()
    g = R.Graph(lambda s: call(b, stream=s, bufs=d))
    for step in range(4):
        b["index"] = R.i32(b["index"] + 1)
        b["pos"] = R.i32((b["pos"] + 17) % b["npos"])
        b["x"] = b["rng"].standard_normal(b["x"].shape).astype(np.float32)
        k, v = b["pool"].download()
        b["pool"].k, b["pool"].v = np.ascontiguousarray(k), np.ascontiguousarray(v)
        for name in ("index", "pos", "x"):
            d[name].upload(b[name])
        g.replay()
        check(b, d, ldo)
    g.close()
