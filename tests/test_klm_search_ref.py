"""The float64 decoder and search that the device's beam search is compared with:
the decoder against the oracle, and the distance between what a search takes and
what it leaves, without which a comparison of tokens would say nothing."""
import numpy as np
import pytest

import klm_search_ref as S
import oracle as O


@pytest.fixture(scope="module")
def weights():
    return S.weights()


@pytest.mark.parametrize("qk_norm", [False, True])
def test_decoder_is_the_oracles(weights, qk_norm):
    """f32 sums of at most 512 terms against float64: 3e-5 of the terms' sum, which
    random signs leave at about 3e-6 of logits up to ten"""
    o = O.CausalLM(S.TINY, qk_norm=qk_norm)
    emb, layers, head = weights
    o.set_embed(emb)
    for i, projs in enumerate(layers):
        for p, b in enumerate(projs):
            o.set_proj(i, p, "q4_k" if p < 6 else "q6_k", b)
    o.set_lm_head("q6_k", head)
    m = S.Model(weights, qk_norm=qk_norm)
    ids = O.token_ids(11, 77, S.TINY["vocab"])
    got, ks, vs = m.prefill(ids)
    assert np.abs(got - o.prefill(ids)).max() <= 3e-4
    for t in (3, 200, 41, 7):
        got, ks, vs = m.step(np.array([t]), len(ids), ks, vs)
        ids = np.append(ids, t)
        assert np.abs(got[0] - o.forward_one(t)).max() <= 3e-4


@pytest.mark.parametrize("case", S.CASES, ids=str)
def test_choices_are_apart(weights, case):
    W, _, max_new, kv, qk_norm, _, eos, bound = case
    beams, gap, early = S.search(S.Model(weights, qk_norm=qk_norm, kv=kv), S.prompt_of(case), max_new, W, eos)
    assert gap >= 2 * bound and len(beams) == W
    assert eos < 0 or early >= 1  # beams end before the others
