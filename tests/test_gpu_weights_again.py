"""Decoders whose weights are set again between calls: every result is that of a
decoder that got them first, whatever step was captured before."""
import numpy as np
import pytest

import oracle as O
from synapse_amd import hip

pytestmark = pytest.mark.gpu
INT8 = dict(hidden=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, inter=512, vocab=384, max_seq=64)
HYBRID = dict(hidden=256, n_layers=4, vocab=512, n_heads=4, n_kv_heads=2, head_dim=64, inner=256,
              conv_kernel=3, inter=512, max_seq=96, eps=1e-5, rope_theta=1e4, layer_kinds=[0, 1, 0, 1])
MAMBA = dict(d_model=64, d_inner=128, d_state=16, d_conv=4, dt_rank=8, n_layers=2, vocab=256, max_tokens=64)
PROMPT = O.token_ids(9, 3, 256)
NAMES = ("q", "k", "v", "o", "gate", "up", "down")


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


def same(a, b):
    for x, y in zip(a, b):
        assert np.array_equal(x, y)


def int8_layer(seed):
    h, qd, kvd, inter = 256, 256, 128, 512
    shapes = [(qd, h), (kvd, h), (kvd, h), (h, qd), (inter, h), (inter, h), (h, inter)]
    return [O.normal(r * c, seed + i, 0.05).reshape(r, c) for i, (r, c) in enumerate(shapes)]


def int8(seeds=(100, 200), embed=1):
    m = hip.QuantizedCausalLM(INT8)
    m.set_weights(O.normal(384 * 256, embed, 0.05).reshape(384, 256),
                  [dict(zip(NAMES, int8_layer(s))) for s in seeds],
                  lm_head=O.normal(384 * 256, 2, 0.05).reshape(384, 256))
    return m


def int8_results(m):
    return [*m.generate(PROMPT, 12), m.prefill(PROMPT), m.forward_one(5)]


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("graph", [True, False])
def test_int8_layer_and_embedding_again(fused, graph):
    m = int8()
    m.set_options(fused, graph)
    first = int8_results(m)
    arrs = int8_layer(300)
    hip.check(hip.lib().syn_hip_qlm_set_layer(m.h, 1, *[hip.ptr(a) for a in arrs]))
    now, want = int8_results(m), int8((100, 300))
    want.set_options(fused, graph)
    same(now, int8_results(want))
    assert not np.array_equal(now[-1], first[-1])
    e = O.normal(384 * 256, 7, 0.05).reshape(384, 256)
    hip.check(hip.lib().syn_hip_qlm_set_embed(m.h, hip.ptr(e)))
    want = int8((100, 300), embed=7)
    want.set_options(fused, graph)
    same(int8_results(m), int8_results(want))


@pytest.mark.parametrize("kind", ["int8", "hybrid", "mamba", "mamba_xdt"])
def test_synthetic_weights_again(kind):
    make = {"int8": lambda: hip.QuantizedCausalLM(INT8), "hybrid": lambda: hip.HybridLM(HYBRID),
            "mamba": lambda: hip.QuantizedMamba(MAMBA),
            "mamba_xdt": lambda: hip.QuantizedMamba(MAMBA, int8_xdt=True)}[kind]
    m = make()
    for seed in (0x5EED0000, 0x5EED4000, 0x5EED0000):
        m.init_synthetic(seed, 0.06)
        want = make()
        want.init_synthetic(seed, 0.06)
        for _ in range(2):
            same(m.generate(PROMPT, 12), want.generate(PROMPT, 12))
