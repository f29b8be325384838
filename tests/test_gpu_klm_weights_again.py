"""A K-quant decoder whose weights are set again between calls: every result is
that of a decoder that got them first, whatever steps were captured before."""
import numpy as np
import pytest

import oracle as O
from synapse_amd import hip
from test_gpu_klm_beams import TINY, build

pytestmark = pytest.mark.gpu
F4, F6 = hip.FMT_Q4_K, hip.FMT_Q6_K
H, QD, KVD, INTER = TINY["hidden"], 256, 128, TINY["inter"]
SHAPES = [(QD, H, F4), (KVD, H, F4), (KVD, H, F4), (H, QD, F4), (INTER, H, F4), (INTER, H, F4), (H, INTER, F6)]
PROMPT = O.token_ids(20, 4, TINY["vocab"])


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


def everything(g):
    """the decoder's captured steps (greedy, draft, beams) and its eager ones"""
    out = list(g.generate(PROMPT, 12))
    out += list(g.generate_speculative(PROMPT, 12, 2, 1))
    out += list(g.generate_beams(PROMPT, 9, 4))
    out += [g.prefill(PROMPT), g.forward_one(3)]
    return out


def same(a, b):
    for x, y in zip(a, b):
        assert np.array_equal(x, y)


def proj(p, seed):
    n, k, f = SHAPES[p]
    return hip.kquant_encode(f, O.normal(n * k, seed, 0.06).reshape(n, k))


def embed(seed):
    return O.normal(TINY["vocab"] * H, seed, 0.5).reshape(TINY["vocab"], H)


def head(seed):
    return hip.kquant_encode(F6, O.normal(TINY["vocab"] * H, seed, 0.3).reshape(TINY["vocab"], H))


@pytest.mark.parametrize("finalize", [True, False])
@pytest.mark.parametrize("what", ["embed", "head", "o", "down"])
def test_one_weight_again(what, finalize):
    def change(m):
        if what == "embed":
            m.set_embed(embed(91))
        elif what == "head":
            m.set_lm_head(head(92))
        else:
            m.set_proj(1, 3 if what == "o" else 6, proj(3 if what == "o" else 6, 93))

    _, g = build()
    _, want = build()
    first = everything(g)
    change(g)
    change(want)
    want.finalize()
    if finalize:
        g.finalize()
    same(everything(g), everything(want))
    _, old = build()
    same(first, everything(old))


def test_finalized_twice():
    """the fused step's scratch is new each time"""
    _, g = build()
    first = everything(g)
    g.finalize()
    same(everything(g), first)


@pytest.mark.parametrize("order", [(0, 1, 2, 3, 4, 5, 6), (2, 1, 0, 6, 5, 4, 3), (5, 0, 4, 2, 1)])
@pytest.mark.parametrize("finalize", [True, False])
def test_stacked_projections_again(order, finalize):
    """q, k and v are one matrix, and gate and up: refused while one of them is missing"""
    _, g = build()
    first = everything(g)
    _, want = build()
    for i, p in enumerate(order):
        g.set_proj(0, p, proj(p, 70 + p))
        want.set_proj(0, p, proj(p, 70 + p))
        done = set(order[:i + 1])
        partial = (len(done & {0, 1, 2}) % 3, len(done & {4, 5}) % 2) != (0, 0)
        ids, out = PROMPT.copy(), np.zeros(TINY["vocab"], np.float32)
        call = hip.lib().syn_hip_klm_forward_prefill(g.h, hip.ptr(ids), ids.size, hip.ptr(out))
        assert call == (2 if partial else 0)
        if partial:
            assert hip.lib().syn_hip_klm_finalize(g.h) == 2
    want.finalize()
    if finalize:
        g.finalize()
    now = everything(g)
    same(now, everything(want))
    assert not np.array_equal(now[-1], first[-1])


def test_all_weights_again():
    """as a file loaded a second time sets them"""
    _, g = build()
    first = everything(g)
    for seed in (0x5EED1000, 0x5EED0000):
        _, other = build(seed=seed)
        g.set_embed(O.normal(TINY["vocab"] * H, seed, 0.5).reshape(TINY["vocab"], H))
        for layer in range(TINY["n_layers"]):
            for p in range(7):
                g.set_proj(layer, p, proj(p, seed + 1 + 8 * layer + p))
        w = O.normal(TINY["vocab"] * H, seed + 1 + 8 * TINY["n_layers"], 0.2).reshape(TINY["vocab"], H)
        g.set_lm_head(hip.kquant_encode(F6, w))
        g.finalize()
        same(everything(g), everything(other))
    same(everything(g), first)
