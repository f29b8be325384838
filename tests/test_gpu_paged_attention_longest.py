"""Attention of new tokens over as many positions as a call takes.  Few pages,
named over and over by the table; only the last position is unlike the others: its
score is 60 above theirs, so with 2^31 of them it still has all of the weight of
the last token but 2e-17, and the result is its value to f32's rounding.  The
tokens before it do not see it: theirs is the mean of the others, every weight 1
(sums of some 10^5 tiles in f32, each addition within 2^-24: 1 %)."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from synapse_amd import hip

pytestmark = pytest.mark.gpu
MOST = 0x7fff0000


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


@pytest.mark.parametrize("new,short", [(1, 0), (1, 77), (5, 1), (20, 0), (40, 33)])
@pytest.mark.parametrize("window", [0, 5000, MOST - 100])
def test_longest(new, short, window):
    print("longest", new, short, window, flush=True)
    page, hd, length = 1024, 8, MOST - short
    rng = np.random.default_rng(length)
    pool = R.Pool("f16", page, 3, 1, 1, hd)
    pool.v = R.store(rng.uniform(1, 2, pool.v.shape).astype(np.float32), "f16")
    pool.v[0, 2] = pool.v[0, 0]
    slot = (length - 1) % page
    pool.k[0, 2, 0, slot, 0] = 60
    pool.v[0, 2, 0, slot] = -np.arange(1, hd + 1)
    pool.upload()
    cols = MOST // page
    table = R.i32(np.arange(cols) & 1)
    table[(length - 1) // page] = 2
    q = np.zeros((new, hd), np.float32)
    q[:, 0] = 1
    p = hip.PagedAttention(layer=0, n_heads=1, n_seqs=1, n_tokens=new, max_new=new, max_len=MOST,
                           window=window, scale=1.0, ldq=hd, ldo=hd, ld_table=cols)
    need = C.c_size_t()
    hip.check(hip.lib().syn_hip_paged_attention_workspace(C.byref(pool.desc), C.byref(p), C.byref(need)))
    t, n, dq = R.dev(table), R.dev(R.i32([length])), R.dev(q)
    out, ws = R.dev(np.full((new, hd), 7.0, np.float32)), hip.DeviceBuffer(need.value)
    hip.check(hip.lib().syn_hip_paged_attention(C.byref(pool.desc), C.byref(p), dq.ptr, None, n.ptr, t.ptr,
                                                out.ptr, ws.ptr, need.value, None))
    R.sync()
    got, want = out.download((new, hd), np.float32), -np.arange(1, hd + 1)
    assert (np.abs(got[-1] - want) <= 4 * 2.0 ** -24 * np.abs(want)).all()
    mean = R.values(pool.v, "f16")[0, :2, 0].mean((0, 1))
    # (a window's two ends may cut a page of 1024 positions of 1 to 2: a tenth of 5000's mean at most)
    assert (np.abs(got[:-1] - mean) <= (0.1 if window == 5000 else 0.02) * mean).all()
