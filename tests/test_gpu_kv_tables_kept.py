"""Pages that no row names but the caller keeps by a count of its own, moved to
another pool."""
import ctypes as C

import numpy as np
import pytest

import drafts_ref as D
import paged_ref as R
from synapse_amd import hip
from test_gpu_kv_tables import Device, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


def moved(rows, pages, to_pages):
    """a pool with kept pages and its tables of `rows` rows that hold none, compacted"""
    rng = np.random.default_rng(pages)
    ref, to = D.Tables(16, pages, rows, 3), D.Tables(16, to_pages, rows, 3)
    ref.refs[rng.random(pages) < 0.3] = 2
    pool = R.Pool("f16", 16, pages, 2, 1, 16, rng=rng)
    other = R.Pool("f16", 16, to_pages, 2, 1, 16, fill=3.0)
    to.table[:], to.held[:], to.refs[:] = 99, 99, 99
    dev, into, live = Device(ref), Device(to), R.dev(np.full(1, -5, np.int32))
    hip.check(hip.lib().syn_hip_kv_compact(C.byref(pool.desc), C.byref(dev.desc), C.byref(other.desc),
                                           C.byref(into.desc), live.ptr, dev.ws.ptr, dev.need, None))
    R.sync()
    return ref, to, pool, other, dev, into, live.download((1,), np.int32)[0]


@pytest.mark.parametrize("pages,to_pages", [(40, 40), (70000, 30000)])
def test_a_row_that_holds_nothing_moves_what_is_kept(pages, to_pages):
    ref, to, pool, other, dev, into, live = moved(1, pages, to_pages)
    n, moves = ref.compact(to)
    assert live == n > 0 and len(moves) == min(n, to_pages)
    dev.check()
    into.check()
    for a, b in moves:
        other.k[:, b], other.v[:, b] = pool.k[:, a], pool.v[:, a]
    same(other, [])


def test_tables_without_rows_are_left_alone():
    ref, to, pool, other, dev, into, live = moved(0, 40, 40)
    assert live == -5
    assert (into.b["refs"].download((40,), np.int32) == 99).all()
    same(other, [])
