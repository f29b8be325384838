"""Samples drawn with drafts by the K-quant decoder: the tokens are those of the
definition in float64 (klm_samples_ref.py, whose cases have no decision near a
border), greedy samples those of greedy decoding, and many samples distributed as
the model's own probabilities say."""
import numpy as np
import pytest

import drafts_ref as D
import klm_samples_ref as K
import klm_search_ref as S
import oracle as O
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
@pytest.mark.parametrize("case", K.CASES, ids=str)
def test_tokens(weights, case, graph):
    print("case", case, flush=True)
    n, k, layers, _, max_new, kv, qk_norm, heat, eos, seed = case
    want, rounds, near = K.run(weights, case)
    assert near >= K.bound(case)
    g = S.device_model(weights, qk_norm=qk_norm)
    g.set_options(True, graph)
    toks, lens, ran = g.generate_samples(K.prompt_of(case), max_new, n, k, layers, heat, eos, KV[kv], seed)
    assert lens.tolist() == [len(t) for t in want]
    for t, m, w in zip(toks, lens, want):
        assert t[:m].tolist() == w and (t[m:] == max(eos, 0)).all()
    assert ran >= rounds  # (whether all have ended is looked at now and then)


@pytest.mark.parametrize("case", [c for c in K.CASES if c[7] > 0 and c[0] < 3][:3], ids=str)
def test_a_sample_ends_with_eos(weights, case):
    """the same tokens, cut at one that a sample has in its middle"""
    n, k, layers, _, max_new, kv, qk_norm, heat, _, seed = case
    want, _, _ = K.run(weights, case)
    eos = want[0][len(want[0]) // 2]
    cut = [t[:t.index(eos) + 1] if eos in t else t for t in want]
    g = S.device_model(weights, qk_norm=qk_norm)
    toks, lens, _ = g.generate_samples(K.prompt_of(case), max_new, n, k, layers, heat, eos, KV[kv], seed)
    for t, m, w in zip(toks, lens, cut):
        assert m == len(w) and t[:m].tolist() == w and (t[m:] == eos).all()


def test_all_layers_draft_what_the_model_says(weights):
    """greedy drafts of the whole model are all accepted: five tokens a round"""
    g = S.device_model(weights)
    prompt = O.token_ids(7, 11, 301)
    toks, lens, rounds = g.generate_samples(prompt, 41, 1, 4, S.TINY["n_layers"], 0.0)
    greedy, margins = g.generate(prompt, 41)
    n = 41 if (margins > 2 * S.F32).all() else int(np.argmin(margins > 2 * S.F32))
    assert n >= 5 and toks[0, :n].tolist() == greedy[:n].tolist()
    if n == 41:
        assert rounds == 8


def test_calls_repeat_and_shapes_change(weights):
    g = S.device_model(weights)
    prompt = O.token_ids(9, 12, 301)
    a = g.generate_samples(prompt, 20, 4, 3, 1, 0.8, seed=5)
    b = g.generate_samples(prompt, 20, 4, 3, 1, 0.8, seed=5)
    c = g.generate_samples(prompt, 20, 4, 3, 1, 0.8, seed=6)
    g.generate_beams(prompt, 8, 40)                       # (more rows through the head than before)
    d = g.generate_samples(prompt[:3], 7, 20, 2, 2, 0.5, eos=4, kv_dtype=hip.KV_F16, seed=7)
    beams = g.generate_beams(prompt, 8, 40)
    e = g.generate_samples(prompt, 20, 4, 3, 1, 0.8, seed=5)
    assert (a[0] == b[0]).all() and (a[0] == e[0]).all() and not (a[0] == c[0]).all()
    assert (g.generate_samples(prompt[:3], 7, 20, 2, 2, 0.5, eos=4, kv_dtype=hip.KV_F16, seed=7)[0] == d[0]).all()
    assert (g.generate_beams(prompt, 8, 40)[0] == beams[0]).all()
    assert len({tuple(t) for t in a[0].tolist()}) > 1
    assert g.cache_len() == 9
    greedy = g.generate(prompt, 20)[0]
    assert (greedy == S.device_model(weights).generate(prompt, 20)[0]).all()


def test_weights_set_again(weights):
    other = S.weights(seed=0x5EED0077)
    g = S.device_model(weights)
    prompt = O.token_ids(6, 13, 301)
    g.generate_samples(prompt, 12, 2, 2, 1, 0.7, seed=1)
    g.set_lm_head(other[2])
    g.set_embed(other[0])
    got = g.generate_samples(prompt, 12, 2, 2, 1, 0.7, seed=1)[0]
    fresh = S.device_model((other[0], weights[1], other[2]))
    assert (got == fresh.generate_samples(prompt, 12, 2, 2, 1, 0.7, seed=1)[0]).all()


@pytest.mark.parametrize("k,layers", [(0, 1), (1, 1), (3, 1), (2, 2)])
def test_shares_of_many_samples(weights, k, layers):
    """the pairs of first tokens of 1280 samples against the model's probabilities: each share
    within 5 standard deviations and the bound of a probability (a logit is off by ROWS at most)"""
    cfg = dict(S.TINY, max_seq=256)
    heat, runs = 0.25, 20
    g = S.device_model(weights, cfg)
    prompt = O.token_ids(5, 14, 301)
    pairs = {}
    for seed in range(runs):
        toks, lens, _ = g.generate_samples(prompt, 3, 64, k, layers, heat, seed=100 + seed)
        assert (lens == 3).all()
        for t in toks:
            pairs[(t[0], t[1])] = pairs.get((t[0], t[1]), 0) + 1
    total = 64 * runs
    m = S.Model(weights, cfg)
    first, ks, vs = m.prefill(prompt)
    p = D.softmax(first, heat)
    assert sum(pairs.values()) == total
    for t in np.argsort(-p)[:6]:
        x, _, _ = m.step(np.array([t]), len(prompt), ks, vs)
        q = p[t] * D.softmax(x[0], heat)
        for y in np.argsort(-q)[:4]:
            share = pairs.get((t, y), 0) / total
            assert abs(share - q[y]) <= 5 * np.sqrt(q[y] * (1 - q[y]) / total) + q[y] * 4 * S.ROWS / heat, (t, y, share, q[y])


def test_refusals(weights):
    g = S.device_model(weights)
    prompt = O.token_ids(8, 15, 301)
    ok = dict(max_new=6, n_samples=2, n_draft=2)
    for kw in (dict(n_samples=0), dict(n_samples=65), dict(n_draft=17), dict(n_samples=33, n_draft=2),
               dict(max_new=90), dict(max_new=88, n_draft=2), dict(eos=301), dict(draft_layers=3),
               dict(kv_dtype=3)):
        with pytest.raises(hip.SynapseError):
            g.generate_samples(prompt, **{**ok, **kw})
    with pytest.raises(hip.SynapseError):
        g.generate_samples(prompt[:0], **ok)
    with pytest.raises(hip.SynapseError):
        g.generate_samples(O.token_ids(96, 1, 301), **ok)
    toks, lens, rounds = g.generate_samples(prompt, 87, 2, 2)  # as long as may be
    assert (lens == 87).all() and rounds >= 29
    toks, lens, rounds = g.generate_samples(prompt, 1, 5, 2)
    assert toks.shape == (5, 1) and rounds == 0
    assert (toks == g.generate_samples(prompt, 3, 5, 2)[0][:, :1]).all()
