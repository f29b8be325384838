"""Rows that continue a row that is not its own parent: they stay."""
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


@pytest.mark.parametrize("rows", [7, 1100])
def test_parents_that_are_not_their_own(rows):
    """a parent whose own parent is outside the rows, or another row, is not continued"""
    ref = D.Tables(8, 20 * rows, rows, 4)
    pool = R.Pool("f16", 8, 20 * rows, 1, 1, 8, rng=np.random.default_rng(1))
    ref.resize([20] * rows)
    dev = Device(ref)
    parent = np.arange(rows)
    parent[:7] = [-1, 0, rows, 2, 4, 4, 5]  # 1 of 0 (outside), 3 of 2 (outside), 5 of 4, 6 of 5 (another's)
    parent, lens = R.i32(parent), R.i32([20, 9, 20, 9, 20, 9, 9] + [0] * (rows - 7))
    table = ref.table.copy()
    dev.fork(pool, R.dev(parent), R.dev(lens))
    R.sync()
    copies = ref.fork(parent, lens)
    assert (ref.table[[0, 1, 2, 3, 4, 6]] == table[[0, 1, 2, 3, 4, 6]]).all() and len(copies) == 1
    dev.check()
    same(pool, copies)
