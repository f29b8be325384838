"""Samples and beams of no tokens: checked as any call, lengths, rounds and scores of 0."""
import ctypes as C

import numpy as np
import pytest

import klm_search_ref as S
import oracle as O
from synapse_amd import hip

pytestmark = pytest.mark.gpu
OK, ARG = 0, 2


@pytest.fixture(scope="module")
def model():
    hip.init(0)
    return S.device_model(S.weights())


def samples(g, n_prompt=8, max_new=0, lengths=True, **kw):
    d = dict(n_samples=3, n_draft=2, draft_layers=0, eos=-1, kv_dtype=hip.KV_F32, temperature=1.0, seed=0)
    d.update(kw)
    prompt = O.token_ids(max(n_prompt, 1), 15, 301)
    toks, lens, rounds = np.full((64, 4), 9, np.uint32), np.full(64, 9, np.uint32), C.c_uint32(9)
    st = hip.lib().syn_hip_klm_generate_samples(
        g.h, hip.ptr(prompt), n_prompt, max_new, C.byref(hip.DraftSampling(**d)), hip.ptr(toks),
        hip.ptr(lens) if lengths else None, C.byref(rounds) if lengths else None)
    return st, toks, lens.tolist(), rounds.value


def test_samples_of_no_tokens(model):
    st, toks, lens, rounds = samples(model)
    assert st == OK and lens == [0] * 3 + [9] * 61 and rounds == 0 and (toks == 9).all()
    assert samples(model, lengths=False)[0] == OK
    assert samples(model, n_prompt=96, n_draft=0)[0] == OK
    st, toks, lens, rounds = samples(model, max_new=1)  # ... and then of one
    assert st == OK and lens[:3] == [1] * 3 and rounds == 0


@pytest.mark.parametrize("kw", [dict(n_samples=0), dict(n_samples=65), dict(n_draft=17), dict(n_prompt=0),
                                dict(n_prompt=97), dict(n_prompt=95), dict(eos=301), dict(draft_layers=3),
                                dict(kv_dtype=3)])
def test_refusals_of_samples(model, kw):
    st, toks, lens, rounds = samples(model, **kw)
    assert st == ARG and (toks == 9).all() and lens == [9] * 64 and rounds == 9


def beams(g, n_prompt=8, max_new=0, results=True, **kw):
    d = dict(n_beams=3, eos=-1, kv_dtype=hip.KV_F32, length_penalty=0.0)
    d.update(kw)
    prompt = O.token_ids(max(n_prompt, 1), 15, 301)
    toks, lens, scores = np.full((64, 4), 9, np.uint32), np.full(64, 9, np.uint32), np.full(64, 9, np.float32)
    st = hip.lib().syn_hip_klm_generate_beams(
        g.h, hip.ptr(prompt), n_prompt, max_new, C.byref(hip.BeamSearch(**d)), hip.ptr(toks),
        hip.ptr(lens) if results else None, hip.ptr(scores) if results else None)
    return st, toks, lens.tolist(), scores.tolist()


def test_beams_of_no_tokens(model):
    st, toks, lens, scores = beams(model)
    assert st == OK and lens == scores == [0] * 3 + [9] * 61 and (toks == 9).all()
    assert beams(model, results=False)[0] == OK
    assert beams(model, n_prompt=96)[0] == OK
    st, toks, lens, scores = beams(model, max_new=1)
    assert st == OK and lens[:3] == [1] * 3 and max(scores[:3]) < 0


@pytest.mark.parametrize("kw", [dict(n_beams=0), dict(n_beams=65), dict(n_prompt=0), dict(n_prompt=97),
                                dict(eos=301), dict(kv_dtype=3), dict(length_penalty=float("nan"))])
def test_refusals_of_beams(model, kw):
    st, toks, lens, scores = beams(model, **kw)
    assert st == ARG and (toks == 9).all() and lens == scores == [9] * 64
