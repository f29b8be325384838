"""Samples drawn with drafts, in float64 over klm_search_ref.py's decoder, for the
tests."""
import copy

import numpy as np

import drafts_ref as D
import klm_search_ref as S
from synapse_amd import hip


def draws(seed, n):
    import ctypes as C
    out = np.zeros(n, np.float32)
    hip.check(hip.lib().syn_hip_stdrng_f32(C.c_uint64(seed), n, hip.ptr(out)))
    return out


def samples(model, prompt, max_new, n, k, layers, heat, eos, seed):
    """([tokens of each], rounds, the least distance of a decision from its border)"""
    small = copy.copy(model)
    small.c = dict(model.c, n_layers=layers)
    u = draws(seed, n + max_new * n * (2 * k + 1))
    first, ks0, vs0 = model.prefill(prompt)
    near, got, most = np.inf, [], 0
    greedy = not heat > 0

    def verify(target, draft, drafted, us):
        nonlocal near
        t, m, _, d = D.verify(np.asarray(target), draft, drafted, len(drafted), heat, us, 0, len(drafted))
        near = min(near, d)
        if greedy:  # (a gap of logits)
            for row in target[:m]:
                two = np.sort(row)[-2:]
                near = min(near, two[1] - two[0])
        return [int(x) for x in t[:m]]

    for s in range(n):
        toks = verify([first], None, [], [u[s]])
        ks, vs, rounds = ks0, vs0, 0
        ended = lambda: len(toks) >= max_new or toks[-1] == eos
        while not ended():
            us = u[n + (rounds * n + s) * (2 * k + 1):][:2 * k + 1]
            pos = len(prompt) + len(toks) - 1
            dk, dv, t, drafted, rows = ks[:layers], vs[:layers], toks[-1], [], []
            for i in range(k):
                x, dk, dv = small.step(np.array([t]), pos + i, dk, dv)
                t = verify([x[0]], None, [], [us[i]])[0]
                drafted.append(t)
                rows.append(x[0])
            target, fk, fv, at = [], ks, vs, []
            for i, t in enumerate([toks[-1]] + drafted):
                x, fk, fv = model.step(np.array([t]), pos + i, fk, fv)
                target.append(x[0])
                at.append((fk, fv))
            new = verify(target, np.asarray(rows) if k else None, drafted, us[k:])
            ks, vs = at[len(new) - 1]
            rounds += 1
            for x in new:
                if ended():
                    break
                toks.append(x)
        got.append(toks)
        most = max(most, rounds)
    return got, most, near


# A logit of the device is off by at most delta (klm_search_ref.py's bounds: F32,
# PAGES of 16 bits, ROWS where more than 8 rows go through a product together):
# every probability moves by a factor within e^(2 delta / heat) of 1, an
# acceptance's two sides by two of them, a border of a draw by as much of the
# whole.  So with no decision nearer than 4 delta / heat the tokens are the same.
# (Greedy: a gap of logits above 2 delta.)
# samples, drafts, draft layers, prompt length, new tokens, pages, head norms, heat, eos, seed
CASES = [
    (1, 0, 1, 8, 12, "f32", False, 0.5, -1, 15),
    (1, 2, 2, 4, 14, "f32", False, 1.0, -1, 116),
    (1, 1, 2, 1, 12, "f32", True, 0.8, -1, 0),
    (2, 0, 1, 5, 8, "f32", True, 0.3, -1, 0),
    (2, 3, 1, 8, 10, "f32", False, 0.5, -1, 590),
    (2, 3, 2, 7, 8, "f32", True, 1.0, -1, 52),
    (4, 1, 1, 6, 6, "f32", False, 0.4, -1, 8),
    (1, 2, 1, 8, 4, "f16", True, 0.7, -1, 50),
    (2, 1, 1, 7, 3, "bf16", False, 1.0, -1, 1240),
    (2, 3, 1, 8, 20, "f32", False, 0.0, -1, 0),
    (8, 0, 1, 3, 10, "f32", False, 0.0, -1, 0),
    (16, 3, 1, 40, 12, "f32", True, 0.0, -1, 19),
    (2, 2, 1, 16, 20, "f16", True, 0.0, -1, 1),
]


def bound(case):
    n, k, _, length, _, kv, _, heat = case[:8]
    delta = S.ROWS if max(length, n * (k + 1)) > 8 else (S.F32 if kv == "f32" else S.PAGES)
    return 4 * delta / heat if heat > 0 else 2 * delta


def prompt_of(case):
    import oracle as O
    return O.token_ids(case[3], 0x5EED0000 + case[9], S.TINY["vocab"])


def run(weights, case):
    n, k, layers, _, max_new, kv, qk_norm, heat, eos, seed = case
    return samples(S.Model(weights, qk_norm=qk_norm, kv=kv), prompt_of(case), max_new, n, k, layers, heat, eos,
                   seed)
