"""Sizes at the beam decoding operators' limits: every check comes before the
device is touched, so these run without a GPU."""
import ctypes as C

import pytest

from synapse_amd import hip

OK, ARG = 0, 2
FAKE = 1 << 20  # an aligned address that no refused call may read


def attention_workspace(**kw):
    d = dict(layer=0, n_heads=2, n_groups=1, group_size=1, max_prefix=64, max_suffix=64, scale=0.0,
             ldq=1 << 16, ldo=1 << 16, ld_prefix_table=1 << 28, ld_table=1 << 28)
    d.update(kw)
    pages = hip.KvPages(hip.KV_F16, 16, 8, 1, 2, 8, FAKE, FAKE)
    need = C.c_size_t()
    return hip.lib().syn_hip_prefix_attention_workspace(C.byref(pages), C.byref(hip.PrefixAttention(**d)),
                                                        C.byref(need))


@pytest.mark.parametrize("which", ["max_prefix", "max_suffix"])
@pytest.mark.parametrize("length,want", [(0x7fff0000, OK), (0x7fff0001, ARG), (0x7fffff00, ARG)])
@pytest.mark.parametrize("members", [1, 64])
def test_attention_lengths(which, length, want, members):
    """kernels step past a length, by less than 2^16, in 32 bits"""
    assert attention_workspace(**{which: length}, group_size=members) == want


@pytest.mark.parametrize("chunks,want", [(262136, OK), (262137, ARG), (262143, ARG)])
def test_select_candidates(chunks, want):
    """64 beams, 128 of each chunk: 2^31 - 2^16 places, which the join steps over
    by 1024 in 32 bits"""
    p = hip.BeamSelect(n_groups=1, n_beams=64, n_select=128, eos=0, pad=0, vocab=2048 * chunks,
                       ld_logits=2048 * chunks)
    assert hip.lib().syn_hip_beam_select_workspace(C.byref(p), C.byref(C.c_size_t())) == want


def test_append_without_positions():
    """every token is skipped: nothing is launched that would read a row of empty tables"""
    pages = hip.KvPages(hip.KV_F16, 16, 8, 1, 2, 8, FAKE, FAKE)
    p = hip.KvAppend(layer=0, n_heads=2, n_seqs=1, rotary_dim=8, interleaved=0, n_positions=0, eps=0,
                     ldq=32, ldk=32, ldv=32, ldo=16, ld_table=1)
    assert hip.lib().syn_hip_kv_append(C.byref(pages), C.byref(p), 3, FAKE, FAKE, FAKE, None, None, FAKE,
                                       FAKE, FAKE, None, FAKE, FAKE, 2 * FAKE, None) == OK
