"""Attention over as many positions as a call takes.  Few pages, named over and
over by the table; only the last position is unlike the others: its score is 60
above theirs, so with 2^31 of them it still has all of the weight but 2e-17, and
the result is its value to f32's rounding (a part that is left out or begins
elsewhere gives the others' mean)."""
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


@pytest.mark.parametrize("members", [1, 20, 40])
@pytest.mark.parametrize("short", [0, 1, 77])
def test_longest_prefix(members, short):
    longest(members, MOST - short, True)


@pytest.mark.parametrize("short", [0, 33])
def test_longest_suffix(short):
    longest(1, MOST - short, False)


def longest(members, length, prefix):
    page, hd = 1024, 8
    rng = np.random.default_rng(length)
    pool = R.Pool("f16", page, 3, 1, 1, hd)
    pool.v = R.store(rng.uniform(1, 2, pool.v.shape).astype(np.float32), "f16")
    slot = (length - 1) % page
    pool.k[0, 2, 0, slot, 0] = 60
    pool.v[0, 2, 0, slot] = -np.arange(1, hd + 1)
    pool.upload()
    cols = MOST // page
    table = R.i32(np.arange(cols) & 1)
    table[(length - 1) // page] = 2
    q = np.zeros((members, hd), np.float32)
    q[:, 0] = 1
    none = dict(max_prefix=0, max_suffix=0, ld_prefix_table=0, ld_table=0)
    one = dict(max_prefix=MOST, ld_prefix_table=cols) if prefix else dict(max_suffix=MOST, ld_table=cols)
    p = hip.PrefixAttention(**{**dict(layer=0, n_heads=1, n_groups=1, group_size=members, scale=1.0, ldq=hd,
                                      ldo=hd), **none, **one})
    need = C.c_size_t()
    hip.check(hip.lib().syn_hip_prefix_attention_workspace(C.byref(pool.desc), C.byref(p), C.byref(need)))
    t, n, dq = R.dev(table), R.dev(R.i32([length])), R.dev(q)
    out, ws = R.dev(np.full((members, hd), 7.0, np.float32)), hip.DeviceBuffer(need.value)
    a = (t.ptr, n.ptr, None, None) if prefix else (None, None, t.ptr, n.ptr)
    hip.check(hip.lib().syn_hip_prefix_attention(C.byref(pool.desc), C.byref(p), dq.ptr, *a, out.ptr, ws.ptr,
                                                 need.value, None))
    R.sync()
    want = -np.arange(1, hd + 1)
    assert (np.abs(out.download((members, hd), np.float32) - want) <= 4 * 2.0 ** -24 * np.abs(want)).all()
