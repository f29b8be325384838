"""The order of beam search's choice where values are equal: the lower beam,
then within a beam the larger logit, then the lower token; zeros of either sign
are equal.  Against that order over values formed in float64."""
import numpy as np
import pytest

import paged_ref as R
from synapse_amd import hip
from test_gpu_beam_select import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


def ordered(x, scores, finished, n, pad):
    """parents and tokens of the n best of one group"""
    w, v = x.shape
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    val = np.full((w, v), -np.inf)
    for b in range(w):
        if finished[b]:
            val[b, pad] = scores[b]
        elif x[b].max() > -np.inf:
            d = x[b] - x[b].max()
            val[b] = scores[b] + (d - np.log(np.exp(d).sum()))
    beam, token = np.divmod(np.arange(w * v), v)
    at = np.lexsort((token, -x.reshape(-1), beam, -val.reshape(-1)))[:n]
    return beam[at], token[at]


def check(c):
    c.call()
    R.sync()
    parent, token, _, _ = c.got()
    for g in range(c.g):
        r = slice(g * c.w, (g + 1) * c.w)
        p, t = ordered(c.x[r], c.scores[r].astype(np.float64), c.fin[r], c.n, c.padtok)
        assert np.array_equal(parent[g], p), (g, parent[g], p)
        assert np.array_equal(token[g], t), (g, token[g], t)


@pytest.mark.parametrize("vocab", [4, 300, 3000, 40000])
@pytest.mark.parametrize("n", [1, 3, 9, 70, 128])
@pytest.mark.parametrize("share", [1e-3, 0.02, 0.6])
def test_zeros_of_either_sign(vocab, n, share):
    """the best logits are zeros, as a mask of 0 and 1 leaves them: few, many, and
    more than a list holds"""
    c = Case(1, 2, 1, min(n, vocab), vocab, finished=False)
    c.x[:] = -np.abs(c.x) - 1
    for row in c.x:
        at = c.rng.permutation(vocab)[:max(2, int(vocab * share))]
        row[at] = np.where(c.rng.random(len(at)) < 0.5, np.float32(0.0), np.float32(-0.0))
    c.x[0, [0, 1]] = np.float32([-0.0, 0.0])
    check(c)


def test_zeros_of_either_sign_in_several_beams():
    c = Case(2, 1, 4, 40, 9000, finished=False)
    c.x[:] = -5.0
    c.x[:, ::500] = np.where(c.rng.random((4, 18)) < 0.5, np.float32(0.0), np.float32(-0.0))
    c.scores[:] = -2.0
    check(c)


@pytest.mark.parametrize("first", [0, 1])
def test_finished_and_live_beams_at_zero(first):
    """a finished beam whose score is -0.0 and a live one that is certain of its word"""
    c = Case(3, 1, 2, 2, 600, finished=False)
    c.fin[first] = 1
    c.scores[first], c.scores[1 - first] = -0.0, 0.0
    c.x[1 - first] = -np.inf
    c.x[1 - first, 77] = 1.5
    check(c)
    c.scores[:] = -c.scores
    c.bufs = None
    check(c)


def tight(c, row, at, large=1e18):
    """logits that differ in f32, next to one so large that their values do not in f64"""
    c.x[row] = -np.inf
    c.x[row, at] = np.float32(1 + np.arange(len(at)) % 7)
    c.x[row, at[len(at) // 2]] = large


@pytest.mark.parametrize("vocab,many", [(50, 20), (9000, 60), (9000, 3000), (40000, 1500)])
@pytest.mark.parametrize("n", [1, 2, 8, 40, 128])
def test_logits_whose_values_are_equal(vocab, many, n):
    """in a chunk, over chunks, and more of them than are ranked at once"""
    c = Case(4, 2, 2, min(n, many), vocab, finished=False)
    for row in range(4):
        tight(c, row, np.sort(c.rng.permutation(vocab)[:many]))
    c.scores[:] = -3.0
    c.scores[3] = -4.0
    check(c)


def test_equal_values_of_beams_live_and_finished():
    """the beams' best words meet at one value"""
    c = Case(5, 1, 5, 10, 2100, finished=False)
    c.fin[[1, 3]] = 1
    for row in (0, 2, 4):
        tight(c, row, np.sort(c.rng.permutation(2100)[:30]), large=1e17)
    c.scores[:] = -3.0
    check(c)


@pytest.mark.parametrize("n", [16, 128])
def test_every_beam_the_same(n):
    """64 beams with equal words and scores: more candidates than are ranked at once"""
    c = Case(6, 1, 64, n, 5000, finished=False)
    c.x[:] = np.where(np.arange(5000) % 11 == 0, 2.0, -1.0)
    c.x[:, 4000] = np.float32(2.0000002)
    c.scores[:] = -7.0
    check(c)
