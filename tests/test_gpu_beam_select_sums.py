"""The log-sum of beam search's values where f32 exponentials do worst: many equal
logits far below the top one, whose arguments are all rounded the same way.
Bound of a value: 2^-24 of it (its rounding to f32) and 2^-18 (a chunk's f32 sum:
2.5 ln 8192 units of 2^-24 for the arguments, 2 for the exponential, 39 for the
additions, 64 in all)."""
import numpy as np
import pytest

import paged_ref as R
from synapse_amd import hip
from test_gpu_beam_select import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


@pytest.mark.parametrize("vocab", [2047, 8192, 20000, 151936])
@pytest.mark.parametrize("seed", range(4))
def test_many_logits_far_below_the_top(vocab, seed):
    c = Case(seed, 24, 8 if vocab < 100000 else 4, 3, vocab, finished=False)
    for row in c.x:  # the others together weigh about as much as the top
        top = np.float32(c.rng.uniform(-9, 9))
        row[:] = top - np.float32(np.log(vocab) + c.rng.uniform(-2, 2))
        row[c.rng.integers(0, vocab, 3)] = top
    c.scores[:] = 0.0
    c.call()
    R.sync()
    parent, token, value, _ = c.got()
    x = c.x.reshape(c.g, c.w, vocab)
    for g in range(c.g):
        for p, t, v in zip(parent[g], token[g], value[g]):
            row = x[g, p].astype(np.float64)
            want = row[t] - row.max() - np.log(np.exp(row - row.max()).sum())
            assert abs(v - want) <= 2.0 ** -24 * abs(want) + 2.0 ** -18
    # (rows whose best values are further apart than the bound are in order)
    for g in range(c.g):
        best = [r.astype(np.float64).max() for r in x[g]]
        lse = [m + np.log(np.exp(r.astype(np.float64) - m).sum()) for m, r in zip(best, x[g])]
        tops = sorted(((b - s) for b, s in zip(best, lse)), reverse=True)
        assert abs(value[g][0] - tops[0]) <= 2.0 ** -17
