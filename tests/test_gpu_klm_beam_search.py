"""The device's beam search against the search in float64, by tokens: pages of
every type, head norms, up to 64 beams, beams that end early.  No choice of a
case is closer than twice the bound of a score (klm_search_ref.py, and
test_klm_search_ref.py asserts it), so the sets of beams are the same."""
import numpy as np
import pytest

import klm_search_ref as S
from synapse_amd import hip

pytestmark = pytest.mark.gpu
KV = {"f32": hip.KV_F32, "f16": hip.KV_F16, "bf16": hip.KV_BF16}


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


@pytest.fixture(scope="module")
def weights():
    return S.weights()


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("case", S.CASES, ids=str)
def test_tokens_of_a_search(weights, case, graph):
    print("case", case, flush=True)
    W, _, max_new, kv, qk_norm, _, eos, bound = case
    prompt = S.prompt_of(case)
    want, gap, _ = S.search(S.Model(weights, qk_norm=qk_norm, kv=kv), prompt, max_new, W, eos)
    assert gap >= 2 * bound
    g = S.device_model(weights, qk_norm=qk_norm)
    g.set_options(True, graph)
    toks, lens, scores = g.generate_beams(prompt, max_new, W, eos, KV[kv])
    got = {tuple(int(x) for x in t[:n]): float(s) for t, n, s in zip(toks, lens, scores)}
    assert got.keys() == want.keys()
    off = max(abs(got[t] - want[t]) for t in got)
    print("scores off by", off)
    assert off <= bound
    assert (np.diff(scores) <= 0).all()
    for t, n in zip(toks, lens):
        assert n == max_new or (t[n - 1:] == eos).all()
