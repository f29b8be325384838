"""Verification of drafted tokens against float64.

Tokens and counts are whole numbers and have to be those of the definition;
each case asserts that no decision of its lies within 2^-30 of a border, 2^10
times what the f64 sums of 150000 terms may be off.  A log-probability is an
f64 value rounded once: 2^-24 of itself, and 2^-40 for the f64 sums."""
import ctypes as C

import numpy as np
import pytest

import drafts_ref as D
import paged_ref as R
from synapse_amd import hip

pytestmark = pytest.mark.gpu
PAD = 77


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


class Case:
    def __init__(self, seed, seqs, drafts, vocab, certain=False, near=0.5, spread=2.5, ld=None, heat=None,
                 step_major=False):
        rng = self.rng = np.random.default_rng(seed)
        self.n, self.d, self.vocab, self.ld = seqs, drafts, vocab, ld or vocab
        self.certain, self.step_major = certain, step_major
        self.draft = (rng.standard_normal((seqs, max(drafts, 1), self.ld)) * spread).astype(np.float32)
        self.target = (rng.standard_normal((seqs, drafts + 1, self.ld)) * spread).astype(np.float32)
        if drafts:
            self.target[:, :drafts] = self.draft[:, :drafts] + near * self.target[:, :drafts] / spread
        self.heat = np.full(seqs, 1.0, np.float32) if heat is None else np.asarray(heat, np.float32)
        self.u = rng.random((seqs, drafts + 1), np.float32)
        self.drafted = np.zeros((seqs, max(drafts, 1)), np.int32)
        for s in range(seqs):
            for i in range(drafts):
                q = D.softmax(self.draft[s, i, :vocab], self.heat[s] if self.heat[s] > 0 else 1.0)
                self.drafted[s, i] = rng.choice(vocab, p=q) if q.sum() > 0.5 else 0
                if not self.heat[s] > 0:
                    self.drafted[s, i] = self.target[s, i, :vocab].argmax()
        self.count = R.i32(rng.integers(0, drafts + 1, seqs))
        self.count[0] = drafts
        self.bufs = None

    def buffers(self, logp=True):
        p = hip.DraftVerify(n_seqs=self.n, max_draft=self.d, pad=PAD, vocab=self.vocab, ld_target=self.ld,
                            target_stride=(self.d + 1) * self.ld, ld_draft=self.ld,
                            draft_stride=max(self.d, 1) * self.ld)
        draft = self.draft
        if self.step_major:  # the draft's rows step by step, all sequences of a step together
            p.ld_draft, p.draft_stride = self.n * self.ld, self.ld
            draft = draft.transpose(1, 0, 2)
        need = C.c_size_t()
        hip.check(hip.lib().syn_hip_draft_verify_workspace(C.byref(p), C.byref(need)))
        self.p, self.need = p, need.value
        self.bufs = dict(target=R.dev(self.target), draft=R.dev(draft), drafted=R.dev(self.drafted),
                         n=R.dev(self.count), heat=R.dev(self.heat), u=R.dev(self.u),
                         token=R.dev(np.full((self.n, self.d + 1), 5, np.int32)),
                         emitted=R.dev(np.full(self.n, 9, np.int32)),
                         logp=R.dev(np.full((self.n, self.d + 1), 3.0, np.float32)) if logp else None,
                         ws=R.dev(np.full(need.value + 256, 0xFF, np.uint8)))

    def call(self, stream=None):
        if self.bufs is None:
            self.buffers()
        b = self.bufs
        at = lambda k: b[k].ptr if b[k] is not None else None
        hip.check(hip.lib().syn_hip_draft_verify(
            C.byref(self.p), at("target"), None if self.certain else at("draft"), at("drafted"), at("n"),
            at("heat"), at("u"), at("token"), at("emitted"), at("logp"), at("ws"), self.need, stream),
            "draft_verify")

    def got(self):
        b = self.bufs
        return (b["token"].download((self.n, self.d + 1), np.int32), b["emitted"].download((self.n,), np.int32),
                b["logp"].download((self.n, self.d + 1), np.float32) if b["logp"] else None)

    def check(self):
        token, emitted, logp = self.got()
        tail = self.bufs["ws"].download((self.need + 256,), np.uint8)[self.need:]
        assert (tail == 0xFF).all()
        for s in range(self.n):
            want, n, lp, near = D.verify(self.target[s, :, :self.vocab],
                                         None if self.certain else self.draft[s, :, :self.vocab],
                                         self.drafted[s].view(np.uint32), int(self.count[s]), self.heat[s],
                                         self.u[s], PAD, self.d)
            assert near > 2.0 ** -30, (s, near)
            assert emitted[s] == n and (token[s] == want).all(), (s, token[s], want, near)
            if logp is not None:
                with np.errstate(invalid="ignore"):
                    assert ((np.abs(logp[s] - lp) <= 2.0 ** -24 * np.abs(lp) + 2.0 ** -40)
                            | (logp[s] == lp)).all(), (s, logp[s], lp)


CASES = [  # sequences, drafts, vocabulary
    (1, 4, 32000), (5, 3, 1000), (3, 1, 1), (4, 2, 2), (2, 8, 70), (7, 5, 8192), (7, 5, 8193), (3, 4, 8191),
    (2, 3, 151936), (1, 64, 300), (6, 0, 32000), (33, 0, 999), (1, 0, 128256), (2, 12, 20011), (300, 2, 50)]


@pytest.mark.parametrize("seqs,drafts,vocab", CASES)
def test_verify(seqs, drafts, vocab):
    print("verify", seqs, drafts, vocab, flush=True)
    heat = np.random.default_rng(vocab).uniform(0.5, 1.5, seqs).astype(np.float32)
    heat[2::5] = 0
    c = Case(vocab + seqs, seqs, drafts, vocab, heat=heat)
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("near", [0.0, 0.05, 3.0])
def test_drafts_that_are_right_or_wrong(near):
    c = Case(21, 24, 6, 5000, near=near)
    c.call()
    R.sync()
    c.check()
    emitted = c.got()[1]
    if near == 0.0:  # the target itself: every draft is accepted (u q < p for u < 1)
        assert (emitted == c.count + 1).all()
    elif near == 3.0:
        assert emitted.mean() < c.count.mean()


@pytest.mark.parametrize("vocab", [600, 40000])
def test_certain_drafts(vocab):
    c = Case(22, 16, 4, vocab, certain=True, spread=6.0)
    c.drafted[::3, 0] = c.target[::3, 0, :vocab].argmax(-1)
    c.call()
    R.sync()
    c.check()


def test_strides_and_order_of_rows():
    for step_major in (False, True):
        c = Case(23, 5, 4, 3001, ld=3007, step_major=step_major)
        c.target[:, :, 3001:] = 1e30  # behind a row
        c.draft[:, :, 3001:] = 1e30
        c.call()
        R.sync()
        c.check()


def test_one_row_for_all_sequences():
    """a target stride of 0: several draws from one row"""
    c = Case(24, 9, 0, 20000)
    c.target[:] = c.target[0]
    c.buffers()
    c.p.target_stride = 0
    c.call()
    R.sync()
    c.check()
    assert len(np.unique(c.got()[0])) > 3


def test_left_out_and_cut_counts():
    c = Case(25, 6, 3, 700)
    c.count = R.i32([-1, 9, 3, -2147483648, 0, 1])
    c.call()
    R.sync()
    c.check()


def test_defaults():
    """no counts: all drafts; no temperatures: 1; no log-probabilities"""
    c = Case(26, 4, 3, 900)
    c.count[:] = 3
    c.buffers(logp=False)
    c.bufs["n"] = c.bufs["heat"] = None
    c.call()
    R.sync()
    c.check()


@pytest.mark.parametrize("vocab", [50, 9000])
def test_masked_and_infinite_logits(vocab):
    """-inf and the type's lowest value at banned tokens, NaN as -inf, rows of -inf alone, +inf"""
    c = Case(27, 12, 3, vocab)
    low = np.finfo(np.float32).min
    c.target[:, :, 1::3] = -np.inf
    c.draft[1::2, :, 1::3] = -np.inf
    c.target[2, :, 2::3] = low
    c.draft[2, :, 2::3] = low
    c.target[3, :, ::7] = np.nan
    c.draft[3, :, ::5] = np.nan
    c.target[4, 0] = -np.inf     # no token at all
    c.target[5, 3] = np.nan
    c.target[6, 0, [4, 9]] = np.inf
    c.draft[6, 0, [9, 12]] = np.inf
    c.draft[7, 0] = -np.inf      # a draft model that says nothing
    c.target[8, :, 6] = np.inf
    c.heat[9:] = 0
    c.target[9, 0] = -np.inf
    c.target[10, 0, [8, 3]] = np.inf
    c.drafted[10, 0] = 3
    c.count[:] = 3
    c.drafted[6, 0] = 9
    c.call()
    R.sync()
    c.check()
    token, emitted, logp = c.got()
    assert emitted[4] == 1 and token[4, 0] == PAD and logp[4, 0] == -np.inf
    assert emitted[9] == 1 and token[9, 0] == PAD and token[10, 0] == 3


def test_temperatures():
    """small and large ones; those that mean greedy"""
    heat = [1e-3, 1e-30, 1e-40, 50.0, 1e30, 3e38, 0.0, -1.0, np.nan, np.inf, -np.inf, -0.0]
    c = Case(28, len(heat), 2, 4000, heat=heat)
    for s in range(6, 12):
        c.drafted[s] = c.target[s, :2].argmax(-1)
    c.call()
    R.sync()
    c.check()


def test_drafts_outside_the_vocabulary():
    c = Case(29, 4, 2, 300)
    c.drafted[:, 0] = [300, -1, 2 ** 31 - 1, -2 ** 31]
    c.count[:] = 2
    c.heat[3] = 0
    c.call()
    R.sync()
    c.check()
    assert (c.got()[1] == 1).all()


def test_nothing_left_of_the_target():
    """q above p at the draft alone, where p is nothing else: the draw falls back on p"""
    c = Case(30, 2, 1, 100)
    c.target[:, 0] = -np.inf
    c.target[:, 0, 40] = 0.0
    c.draft[:] = -np.inf
    c.draft[:, 0, 40] = 0.0
    c.drafted[:] = 40
    c.count[:] = 1
    c.u[0, 0] = 1.0  # (outside [0, 1), the one way to reject a draft that is certain)
    c.call()
    R.sync()
    token, emitted, _ = c.got()
    assert token[0, 0] == 40 and emitted[0] == 1
    assert token[1, 0] == 40 and emitted[1] == 2


def test_ends_of_the_draw():
    """u of 0 takes the first token that has a weight; the largest u one of the last"""
    c = Case(31, 2, 0, 30000, spread=0.1)
    c.target[:, :, :100] = -np.inf
    c.target[:, :, -100:] = -np.inf
    c.u[:, 0] = [0.0, np.float32(1) - np.float32(2 ** -24)]
    c.call()
    R.sync()
    token = c.got()[0][:, 0]
    # (30000 weights of about 2^-15 each: 2^-24 before the end is the last one)
    assert token[0] == 100 and token[1] == 30000 - 101


def test_ties_go_to_the_lowest_token():
    c = Case(32, 3, 1, 20000)
    c.target[:] = 1.0
    c.heat[:] = 0
    c.drafted[:, 0] = [0, 5, 0]
    c.count[:] = 1
    c.call()
    R.sync()
    token, emitted, _ = c.got()
    assert emitted.tolist() == [2, 1, 2] and (token[:, 0] == 0).all() and token[0, 1] == 0


@pytest.mark.parametrize("seqs,drafts", [(1, 0), (2, 3)])
def test_many_blocks(seqs, drafts):
    """a vocabulary of 342 blocks: more chunks and sums than a wave has lanes"""
    c = Case(36, seqs, drafts, 700001)
    c.call()
    R.sync()
    c.check()


def test_captured_and_replayed():
    a, b = Case(33, 6, 4, 9001), Case(34, 3, 2, 500)
    graphs = []
    for c in (a, b):
        c.call()
        R.sync()
        graphs.append(R.Graph(lambda s, c=c: c.call(s)))
    for _ in range(4):
        for c in (a, b):
            c.u = c.rng.random(c.u.shape, np.float32)
            c.count = R.i32(c.rng.integers(-1, c.d + 1, c.n))
            c.bufs["u"].upload(c.u)
            c.bufs["n"].upload(c.count)
        R.sync()
        for g in graphs:
            g.replay()
        for c in (a, b):
            c.check()
    for g in graphs:
        g.close()


def test_shares_over_many_draws():
    """the first token of drafted sequences is distributed as the target (4000 draws of 12 tokens:
    5 standard deviations of each share)"""
    n, vocab = 4000, 12
    c = Case(35, n, 2, vocab)
    c.target[:], c.draft[:] = c.target[0], c.draft[0]
    q = [D.softmax(c.draft[0, i], 1.0) for i in range(2)]
    for i in range(2):
        c.drafted[:, i] = c.rng.choice(vocab, n, p=q[i])
    c.count[:] = 2
    c.call()
    R.sync()
    first = c.got()[0][:, 0]
    p = D.softmax(c.target[0, 0], 1.0)
    share = np.bincount(first, minlength=vocab) / n
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1e-9).all()
