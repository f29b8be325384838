"""The largest vocabulary and the largest tables of the operators for sampling with
drafts, with contents whose results are known without going through them."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from synapse_amd import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


def test_largest_vocabulary():
    """2^31 - 2^20 equal logits: token t for u in [t / V, (t + 1) / V).  The u's lie 2^-6 of a token
    or more from its ends, 2^-37 of the whole, the f64 sums of 2^20 blocks (8192 of them one after
    the other in a lane, each addition within 2^-53) within 2^-40."""
    print("largest vocabulary", flush=True)
    vocab = 0x7ff00000
    row = np.zeros(vocab, np.float32)
    target = hip.DeviceBuffer.from_array(row)
    del row
    u = np.array([0.0, 0.1, 0.5 - 2.0 ** -9, 0.7321, 1 - 2.0 ** -24], np.float32)
    place = u.astype(np.float64) * vocab
    want = np.floor(place).astype(np.int64)
    assert (((place - want > 2.0 ** -6) & (place - want < 1 - 2.0 ** -6)) | (place == want)).all()
    exact = place == want                          # (a border itself: either neighbour)
    n = len(u) + 1
    heat, du = np.full(n, 0.7, np.float32), np.append(u, np.float32(0.5))
    heat[-1] = 0                                   # greedy: the first of the largest
    p = hip.DraftVerify(n_seqs=n, max_draft=0, pad=0, vocab=vocab, ld_target=vocab, target_stride=0)
    need = C.c_size_t()
    hip.check(hip.lib().syn_hip_draft_verify_workspace(C.byref(p), C.byref(need)))
    ws, dh, d = hip.DeviceBuffer(need.value), R.dev(heat), R.dev(du)
    token, count, logp = (R.dev(np.zeros(n, t)) for t in (np.int32, np.int32, np.float32))

    def draw():
        hip.check(hip.lib().syn_hip_draft_verify(C.byref(p), target.ptr, None, None, None, dh.ptr, d.ptr, token.ptr,
                                                 count.ptr, logp.ptr, ws.ptr, need.value, None))
        R.sync()
        return token.download((n,), np.int32).astype(np.int64)

    got = draw()
    off = want - got[:-1]
    assert ((off == 0) | (exact & (off == 1) & (want > 0))).all(), (got, want)
    assert got[-1] == 0 and (count.download((n,), np.int32) == 1).all()
    lp = logp.download((n,), np.float32)
    assert (np.abs(lp[:-1] + np.log(vocab)) <= 2.0 ** -24 * np.log(vocab) + 2.0 ** -40).all() and lp[-1] == 0
    # all of the weight on the last token but one
    one = np.full(1, 100.0, np.float32)
    hip.check(hip.lib().syn_hip_memcpy_h2d(target.ptr + (vocab - 2) * 4, hip.ptr(one), 4))
    got = draw()
    assert got[0] == 0 and (got[1:] == vocab - 2).all()  # (u = 0: the first token that has a weight)


def test_largest_tables():
    """2^24 pages to 65535 rows: taken in order, given back by every other row, taken again"""
    print("largest tables", flush=True)
    page, pages, rows, cols = 8, 1 << 24, 65535, 256
    b = dict(table=R.dev(np.full((rows, cols), -1, np.int32)), held=R.dev(R.i32(np.zeros(rows))),
             refs=R.dev(R.i32(np.zeros(pages))))
    t = hip.KvTables(page, pages, rows, cols, b["table"].ptr, b["held"].ptr, b["refs"].ptr)
    need = C.c_size_t()
    hip.check(hip.lib().syn_hip_kv_tables_workspace(C.byref(t), C.byref(need)))
    ws = hip.DeviceBuffer(need.value)

    def resize(lens):
        d = R.dev(R.i32(lens))
        hip.check(hip.lib().syn_hip_kv_resize(C.byref(t), d.ptr, ws.ptr, need.value, None))
        R.sync()
        return (b["table"].download((rows, cols), np.int32), b["held"].download((rows,), np.int32),
                b["refs"].download((pages,), np.int32))

    table, held, refs = resize(np.full(rows, cols * page))
    full = np.arange(rows * cols, dtype=np.int32).reshape(rows, cols)
    assert (table == full).all() and (held == cols).all()
    assert (refs[:rows * cols] == 1).all() and (refs[rows * cols:] == 0).all()
    odd = np.arange(rows) % 2 == 1
    table, held, refs = resize(np.where(odd, 0, -1))
    assert (table[odd] == -1).all() and (table[~odd] == full[~odd]).all()
    assert (held == np.where(odd, 0, cols)).all() and refs.sum() == (~odd).sum() * cols
    # the odd rows take a page less each, of those that they gave back, lowest first
    table, held, refs = resize(np.where(odd, (cols - 1) * page, -1))
    free = np.concatenate([full[odd].reshape(-1), np.arange(rows * cols, pages)])
    assert (table[odd][:, :-1].reshape(-1) == free[:odd.sum() * (cols - 1)]).all() and (table[odd][:, -1] == -1).all()
    assert (held[odd] == cols - 1).all() and refs.sum() == (~odd).sum() * cols + odd.sum() * (cols - 1)
