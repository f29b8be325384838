"""Drafts from a model that is almost the target.  After a rejected one little is left
of the target, S = sum max(p - q, 0), and the draw's borders are as much less sure:
p and q are within 2^-42 of themselves (exponentials within 2^-43.4, twice), the sums
up to a border and of all within 2^-41 each, so a border within 2^-40 / S of the u's
range.  Each case asserts that no decision is that near to one."""
import numpy as np
import pytest

import drafts_ref as D
import paged_ref as R
from synapse_amd import hip
from test_gpu_draft_verify import PAD, Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


def case(near, vocab):
    c = Case(41, 20, 3, vocab, near=near)
    c.count[:] = 3
    c.u[:, :3] = np.float32(1 - 2.0 ** -24)  # (a draft that the target likes less is rejected)
    return c


def decisions(c):
    """(tokens, count, what is left of the target) of each sequence, and that it is no near thing"""
    for s in range(c.n):
        token, n, _, near = D.verify(c.target[s], c.draft[s], c.drafted[s].view(np.uint32), 3, c.heat[s], c.u[s],
                                     PAD, c.d)
        left = 1.0
        if n <= 3:
            left = np.maximum(D.softmax(c.target[s, n - 1], 1.0) - D.softmax(c.draft[s, n - 1], 1.0), 0).sum()
        assert near > 2.0 ** -39 / left, (s, near, left)
        yield token, n, left


NEAR = [(1e-3, 300), (1e-4, 9000), (1e-5, 160)]


@pytest.mark.parametrize("near,vocab", NEAR)
def test_little_is_left_of_the_target(near, vocab):
    c = case(near, vocab)
    want = list(decisions(c))
    lefts = [left for _, n, left in want if n <= 3]
    assert len(lefts) > 10 and max(lefts) < near
    c.call()
    R.sync()
    token, emitted, _ = c.got()
    for s, (t, n, _) in enumerate(want):
        assert emitted[s] == n and (token[s] == t).all(), s


def test_nothing_is_left_of_rows_that_are_the_same():
    """a draft outside the vocabulary, and rows that are equal: drawn from the target"""
    c = Case(42, 6, 2, 5000)
    c.target[:, :2] = c.draft[:, :2]
    c.drafted[:, 0] = 5000
    c.drafted[3:, 1] = -1
    c.count[:] = 2
    c.call()
    R.sync()
    c.check()
    token, emitted, _ = c.got()
    assert (emitted == 1).all() and len(np.unique(token[:, 0])) > 1
