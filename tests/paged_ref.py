"""Paged caches on the host and the beam decoding operators' definitions in
float64, for the tests."""
import ctypes as C

import numpy as np

from synapse_amd import hip

CODE = {"f32": hip.KV_F32, "f16": hip.KV_F16, "bf16": hip.KV_BF16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def bf16_bits(x):
    """float32 to bfloat16 bits, to nearest even (NaN kept)"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def store(x, dtype):
    """the stored form of float32 values"""
    if dtype == "f32":
        return np.ascontiguousarray(x, np.float32)
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return np.asarray(x, np.float32).astype(np.float16)
    return bf16_bits(np.asarray(x, np.float32))


def values(s, dtype):
    """the float64 values of stored ones"""
    if dtype == "bf16":
        return (s.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return s.astype(np.float64)


class Pool:
    """A pool of pages: host copies in position order, k and v
    [layers][pages][kv][page_size][hd] (stored form), and the device's."""

    def __init__(self, dtype, page, pages, layers, kv, hd, rng=None, fill=None):
        self.dtype, self.page, self.pages, self.layers, self.kv, self.hd = (dtype, page, pages,
                                                                            layers, kv, hd)
        shape = (layers, pages, kv, page, hd)
        if rng is not None:
            self.k = store(rng.standard_normal(shape).astype(np.float32), dtype)
            self.v = store(rng.standard_normal(shape).astype(np.float32), dtype)
        else:
            self.k = store(np.full(shape, 0.0 if fill is None else fill, np.float32), dtype)
            self.v = self.k.copy()
        self.dk = hip.DeviceBuffer.from_array(self.pack_k(self.k))
        self.dv = hip.DeviceBuffer.from_array(self.pack_v(self.v))
        self.desc = hip.KvPages(CODE[dtype], page, pages, layers, kv, hd, self.dk.ptr, self.dv.ptr)

    def pack_k(self, k):
        return np.ascontiguousarray(
            k.reshape(self.layers, self.pages, self.kv, self.page, self.hd // 8, 8)
            .transpose(0, 1, 2, 4, 3, 5))

    def pack_v(self, v):
        return np.ascontiguousarray(
            v.reshape(self.layers, self.pages, self.kv, self.page // 8, 8, self.hd)
            .transpose(0, 1, 2, 3, 5, 4))

    def upload(self):
        self.dk.upload(self.pack_k(self.k))
        self.dv.upload(self.pack_v(self.v))

    def download(self):
        """the device's pools in position order"""
        k = self.dk.download((self.layers, self.pages, self.kv, self.hd // 8, self.page, 8),
                             self.k.dtype)
        v = self.dv.download((self.layers, self.pages, self.kv, self.page // 8, self.hd, 8),
                             self.v.dtype)
        return (k.transpose(0, 1, 2, 4, 3, 5).reshape(self.k.shape),
                v.transpose(0, 1, 2, 3, 5, 4).reshape(self.v.shape))

    def rows(self, which, layer, table, length):
        """[length][kv][hd] float64 of a sequence, NaN where its page is outside the pool"""
        x = values(getattr(self, which)[layer], self.dtype)
        out = np.full((length, self.kv, self.hd), np.nan)
        for i in range(length):
            p = int(table[i // self.page])
            if 0 <= p < self.pages:
                out[i] = x[p, :, i % self.page]
        return out


def dev(a):
    return hip.DeviceBuffer.from_array(np.ascontiguousarray(a))


def i32(a):
    return np.ascontiguousarray(a, np.int32)


def sync():
    hip.check(hip.lib().syn_hip_synchronize())


class Graph:
    """What `record(stream)` launches, captured into a HIP graph."""

    def __init__(self, record):
        hip.lib()
        self.rt = C.CDLL("libamdhip64.so.7")
        self.stream = C.c_void_p()
        hip.check(hip.lib().syn_hip_stream_create(C.byref(self.stream)))
        graph = C.c_void_p()
        assert self.rt.hipStreamBeginCapture(self.stream, 2) == 0  # relaxed
        record(self.stream.value)
        assert self.rt.hipStreamEndCapture(self.stream, C.byref(graph)) == 0
        self.exec = C.c_void_p()
        assert self.rt.hipGraphInstantiate(C.byref(self.exec), graph, None, None, 0) == 0
        assert self.rt.hipGraphDestroy(graph) == 0

    def replay(self):
        assert self.rt.hipGraphLaunch(self.exec, self.stream) == 0
        hip.check(hip.lib().syn_hip_stream_synchronize(self.stream.value))

    def close(self):
        self.rt.hipGraphExecDestroy(self.exec)
        hip.lib().syn_hip_stream_destroy(self.stream.value)


# ---------------------------------------------------------------- definitions
def rotate(x, cos, sin, rd, interleaved):
    """x [..., hd], cos and sin [..., rd / 2]"""
    y = x.copy()
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if interleaved else (x[..., :rd // 2], x[..., rd // 2:rd])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        y[..., 0:rd:2], y[..., 1:rd:2] = ra, rb
    else:
        y[..., :rd // 2], y[..., rd // 2:rd] = ra, rb
    return y


def attention(q, k, v, scale):
    """q [heads][hd], k and v [n][kv][hd] (NaN rows: left out) -> (out, sum of p|v|, max sum |q k|)"""
    heads, hd = q.shape
    kv = k.shape[1]
    keep = ~np.isnan(k[:, 0, 0]) if len(k) else np.zeros(0, bool)
    k, v = k[keep], v[keep]
    out, mag, qk = np.zeros((heads, hd)), np.zeros((heads, hd)), 0.0
    for h in range(heads):
        kk, vv = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        if not len(kk):
            continue
        s = scale * (kk @ q[h])
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], mag[h] = p @ vv, p @ np.abs(vv)
        qk = max(qk, float((np.abs(kk) @ np.abs(q[h])).max()))
    return out, mag, qk


def select(logits, scores, finished, n, eos, pad):
    """one group: logits [beams][vocab] -> parents, tokens, values, finished"""
    w, v = logits.shape
    val = np.full((w, v), -np.inf)
    for b in range(w):
        if not np.isfinite(scores[b]):
            continue
        if finished[b]:
            val[b, pad] = scores[b]
            continue
        x = np.where(np.isnan(logits[b]), -np.inf, logits[b].astype(np.float64))
        top = x.max()
        if top == -np.inf:
            continue
        with np.errstate(invalid="ignore"):
            d = np.where(x == top, 0.0, x - top)
        val[b] = scores[b] + (d - np.log(np.exp(d).sum()))
    order = np.argsort(-val.reshape(-1), kind="stable")[:n]
    parent, token = order // v, order % v
    return parent, token, val.reshape(-1)[order], (finished[parent] != 0) | (token == eos)
