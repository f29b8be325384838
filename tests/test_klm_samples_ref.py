"""The samples that the device's are compared with: no decision of a case lies
nearer to its border than the device's logits may move it."""
import pytest

import klm_samples_ref as K
import klm_search_ref as S


@pytest.fixture(scope="module")
def weights():
    return S.weights()


@pytest.mark.parametrize("case", K.CASES, ids=str)
def test_decisions_are_apart(weights, case):
    got, rounds, near = K.run(weights, case)
    assert near >= K.bound(case)
    n, k, _, _, max_new, _, _, _, eos, _ = case
    assert len(got) == n and all(len(t) == max_new or t[-1] == eos for t in got)
    assert -(-(max_new - 1) // (k + 1)) <= rounds <= max_new - 1
