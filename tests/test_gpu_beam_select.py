"""Beam search's choice against float64: parents, tokens and flags are equal;
a value is off by the rounding to f32 (2^-24 of it) and by the error of the
row's log-sum-exp, whose exponentials are f32 (2^-22 relative each at most, so
2^-22 absolute in the logarithm)."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from synapse_amd import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


class Case:
    def __init__(self, seed, groups, beams, n, vocab, pad=0, eos=2, finished=True, null_flags=False):
        self.rng = np.random.default_rng(seed)
        self.g, self.w, self.n, self.v, self.eos = groups, beams, n, vocab, eos
        self.x = (self.rng.standard_normal((groups * beams, vocab + pad)) * 2.5).astype(np.float32)
        self.scores = (-20 - 3 * self.rng.random(groups * beams)).astype(np.float32)
        self.fin = R.i32(self.rng.random(groups * beams) < 0.3 if finished else
                         np.zeros(groups * beams))
        self.null_flags, self.bufs, self.padtok = null_flags, None, min(eos if eos >= 0 else 0, vocab - 1)

    def params(self):
        return hip.BeamSelect(n_groups=self.g, n_beams=self.w, n_select=self.n, eos=self.eos,
                              pad=self.padtok, vocab=self.v, ld_logits=self.x.shape[1])

    def call(self, stream=None):
        p = self.params()
        if self.bufs is None:
            need = C.c_size_t()
            hip.check(hip.lib().syn_hip_beam_select_workspace(C.byref(p), C.byref(need)))
            self.need = need.value
            out = np.full(self.g * self.n + 5, -7, np.int32)
            self.bufs = dict(x=R.dev(self.x), s=R.dev(self.scores), f=R.dev(self.fin), p=R.dev(out),
                             t=R.dev(out), v=R.dev(out), fo=R.dev(out),
                             ws=R.dev(np.full(need.value + 256, 0xFF, np.uint8)))
        b = self.bufs
        fin = None if self.null_flags else b["f"].ptr
        hip.check(hip.lib().syn_hip_beam_select(C.byref(p), b["x"].ptr, b["s"].ptr, fin, b["p"].ptr,
                                                b["t"].ptr, b["v"].ptr,
                                                None if self.null_flags else b["fo"].ptr,
                                                b["ws"].ptr, self.need, stream), "beam_select")

    def got(self):
        m = self.g * self.n
        r = [self.bufs[k].download((m + 5,), d) for k, d in
             (("p", np.int32), ("t", np.int32), ("v", np.float32), ("fo", np.int32))]
        for a in r:
            assert (a[m:].view(np.int32) == -7).all()
        assert (self.bufs["ws"].download((self.need + 256,), np.uint8)[self.need:] == 0xFF).all()
        return [a[:m].reshape(self.g, self.n) for a in r]

    def check(self):
        parent, token, value, flag = self.got()
        for g in range(self.g):
            r = slice(g * self.w, (g + 1) * self.w)
            fin = np.zeros(self.w, int) if self.null_flags else self.fin[r]
            p, t, v, f = R.select(self.x[r, :self.v], self.scores[r].astype(np.float64), fin, self.n,
                                  self.eos, self.padtok)
            assert np.array_equal(parent[g], p), (g, parent[g], p)
            assert np.array_equal(token[g], t), (g, token[g], t)
            live = np.isfinite(v)
            assert np.array_equal(np.isfinite(value[g]), live)
            assert (value[g][~live] == -np.inf).all()
            assert (np.abs(value[g] - v)[live] <= 2.0 ** -24 * np.abs(v[live]) + 2.0 ** -22).all()
            if not self.null_flags:
                assert np.array_equal(flag[g] != 0, f)


SHAPES = [(1, 4, 4, 32000), (4, 8, 8, 128256), (2, 8, 16, 151936), (3, 1, 1, 1000), (1, 1, 5, 5),
          (2, 3, 12, 4), (1, 64, 128, 2), (2, 64, 64, 3001), (1, 64, 128, 20011), (5, 5, 10, 257),
          (1, 16, 33, 65536), (70, 2, 4, 513), (1, 7, 1, 1)]


@pytest.mark.parametrize("case", SHAPES, ids=str)
def test_select(case):
    print("case", case, flush=True)
    c = Case(1, *case, pad=3 if case[0] % 2 == 0 else 0, finished=case[1] > 1, eos=min(2, case[3] - 1))
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("rows", [3, 64])
@pytest.mark.parametrize("vocab,pad", [(8195, 1), (8196, 4), (30001, 3), (2050, 2), (4, 4), (8198, 0), (8199, 2),
                                       (2055, 0), (4111, 1), (8194, 3)])
def test_rows_that_end_inside_a_chunk(rows, vocab, pad):
    """rows 16 bytes apart, with large values between them"""
    c = Case(11, rows, 2, 4, vocab, pad=pad)
    c.x[:, vocab:] = 100.0
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_logits_that_begin_off_16_bytes(shift):
    c = Case(12, 5, 3, 6, 16390)
    c.call()
    R.sync()
    raw = R.dev(np.concatenate([np.full(shift, 100, np.float32), c.x.reshape(-1)]))

    class Moved:
        ptr = raw.ptr + 4 * shift
    c.bufs["x"] = Moved
    for k in "ptv":
        c.bufs[k] = R.dev(np.full(c.g * c.n + 5, -7, np.int32))
    c.call()
    R.sync()
    c.check()


def test_without_flags_or_eos():
    c = Case(2, 2, 4, 4, 5000, eos=-1, null_flags=True)
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("vocab", [40, 70001])
def test_ties_go_to_the_lowest_index(vocab):
    """equal rows (every beam begins the same) and few different logits"""
    c = Case(3, 2, 4, 16, vocab, finished=False)
    c.x[:4] = c.x[0]
    c.scores[:4] = c.scores[0]
    c.x[4:] = np.round(c.x[4:])
    c.scores[4:] = c.scores[4]
    # the rounded rows hold other sets of logits, so their sums differ; one row repeats
    c.x[6] = c.x[5]
    c.call()
    R.sync()
    c.check()


def test_all_logits_equal():
    c = Case(4, 1, 3, 100, 30000, finished=False)
    c.x[:] = 1.25
    c.scores[:] = np.float32([-3, -3, -2])
    c.call()
    R.sync()
    c.check()


def test_first_step_scores_and_dead_beams():
    """only beam 0 lives; scores of NaN and either infinity have no continuation"""
    c = Case(5, 2, 5, 10, 900, finished=False)
    c.scores[:] = np.float32([-0.0, -np.inf, np.nan, np.inf, -np.inf, np.nan, -np.inf, -1, np.inf, np.nan])
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("w,n,vocab", [(64, 128, 3), (2, 5, 9000)])
def test_no_live_beam_in_a_group(w, n, vocab):
    """the first continuations in order, all of -inf"""
    c = Case(10, 2, w, n, vocab, finished=False)
    c.scores[:w] = -np.inf
    c.call()
    R.sync()
    c.check()


def test_fewer_live_words_than_asked_for():
    c = Case(6, 3, 2, 9, 50, finished=False)
    c.x[0, 3:] = -np.inf
    c.x[1] = -np.inf
    c.x[2:4] = np.nan
    c.x[4, 5:] = -3.4028235e38   # the lowest finite value is a value
    c.x[5, 1:] = np.nan
    c.call()
    R.sync()
    c.check()


def test_infinities_and_nan_among_logits():
    c = Case(7, 2, 3, 6, 20000, finished=False)
    c.x[0, [5, 7000, 19999]] = np.inf
    c.x[1, ::2] = np.nan
    c.x[2, 11] = np.inf
    c.x[3, [0, 19999]] = 3.4028235e38, -3.4028235e38
    c.x[4, :] += 1e30
    c.call()
    R.sync()
    c.check()


def test_finished_beams_with_the_best_and_the_worst_scores():
    c = Case(8, 3, 4, 8, 700)
    c.fin[:] = [1, 0, 0, 0, 1, 1, 1, 1, 0, 7, -1, 0]
    c.scores[[0, 9]] = -1, -500
    c.scores[10] = -np.inf
    c.call()
    R.sync()
    c.check()


def test_pad_at_the_ends_of_a_small_vocabulary():
    for pad in (0, 3):
        c = Case(9, 1, 2, 8, 4, eos=pad)
        c.fin[:] = 1
        c.padtok = pad
        c.call()
        R.sync()
        c.check()


def test_scores_and_flags_in_place_over_replays():
    c = Case(11, 3, 6, 6, 4099)
    c.call()
    R.sync()

    def record(stream):
        p, b = c.params(), c.bufs
        hip.check(hip.lib().syn_hip_beam_select(C.byref(p), b["x"].ptr, b["s"].ptr, b["f"].ptr,
                                                b["p"].ptr, b["t"].ptr, b["s"].ptr, b["f"].ptr,
                                                b["ws"].ptr, c.need, stream))
    g = R.Graph(record)
    for step in range(4):
        c.x = (c.rng.standard_normal(c.x.shape) * 2.5).astype(np.float32)
        c.bufs["x"].upload(c.x)
        R.sync()
        g.replay()
        new = c.bufs["s"].download((18,), np.float32)
        fin = c.bufs["f"].download((18,), np.int32)
        parent = c.bufs["p"].download((18,), np.int32).reshape(3, 6)
        token = c.bufs["t"].download((18,), np.int32).reshape(3, 6)
        for i in range(3):
            r = slice(6 * i, 6 * i + 6)
            p, t, v, f = R.select(c.x[r], c.scores[r].astype(np.float64), c.fin[r], 6, c.eos, c.padtok)
            assert np.array_equal(parent[i], p) and np.array_equal(token[i], t)
            assert (np.abs(new[r] - v) <= 2.0 ** -24 * np.abs(v) + 2.0 ** -22).all()
            assert np.array_equal(fin[r] != 0, f)
        c.scores, c.fin = new, fin
    g.close()


@pytest.mark.parametrize("vocab", [2048, 8192, 30000])
def test_more_equal_logits_than_a_list_holds(vocab):
    """whole chunks of one value, and of a few values with the best repeated"""
    c = Case(12, 2, 3, 7, vocab, finished=False)
    c.x[0] = 0.5
    c.x[1] = np.where(np.arange(vocab) % 3 == 0, 1.0, -1.0)
    c.x[2, vocab // 2:] = -np.inf
    c.x[3:] = np.round(c.x[3:] * 2)
    c.scores[3:] = c.scores[3]
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 128])
def test_few_words_left_by_a_mask(n):
    """most logits are -inf, as a grammar leaves them"""
    c = Case(13, 2, 4, n, 40000, finished=False)
    keep = c.rng.random(c.x.shape) < 2e-3
    c.x[~keep] = -np.inf
    c.x[5] = -np.inf
    c.call()
    R.sync()
    c.check()
