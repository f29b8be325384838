"""The operators for sampling with drafts in the order in which a decoder calls them,
over one attention layer whose queries, keys and values are looked up by token and a
draft model that sees the last token alone.  The host keeps every sample's tokens:
attention is checked against float64 over them (bounds as in
test_gpu_paged_attention.py), drawn and verified tokens against the definition on the
same logits."""
import ctypes as C

import numpy as np
import pytest

import drafts_ref as D
import paged_ref as R
from synapse_amd import hip
from test_gpu_draft_verify import PAD
from test_gpu_paged_attention import causal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rounds_by_hand(dtype):
    rng = np.random.default_rng(8)
    n, K, nh, kv, hd, page, vocab, ldl, rounds, n_prompt = 4, 3, 4, 2, 64, 16, 60, 64, 9, 21
    most = n_prompt + rounds * (K + 1) + K + 1
    cols = -(-most // page)
    pool = R.Pool(dtype, page, n * cols, 1, kv, hd, fill=float("nan"))
    eq, ek, ev = (rng.standard_normal((vocab, w * hd)).astype(np.float32) for w in (nh, kv, kv))
    out_w = rng.standard_normal((nh * hd, vocab)).astype(np.float32)
    draft_w = (rng.standard_normal((vocab, vocab)) * 1.5).astype(np.float32)
    stored = {k: R.values(R.store(v, dtype), dtype).reshape(vocab, kv, hd) for k, v in (("k", ek), ("v", ev))}
    L, heat = hip.lib(), np.full(n, 0.9, np.float32)
    f32, z = np.float32, lambda *s: np.zeros(s, np.float32)
    b = {k: R.dev(v) for k, v in dict(
        table=np.full((n, cols), -1, np.int32), held=R.i32(np.zeros(n)), refs=R.i32(np.zeros(n * cols)),
        heat=heat, ws=np.zeros(1 << 20, np.uint8), x=R.i32(np.zeros(n)), drafted=R.i32(np.zeros((n, K))),
        tokens=R.i32(np.zeros((n, K + 1))), count=R.i32(np.zeros(n)), logits=z(n, K + 1, ldl),
        draft=z(K, n, ldl), u=z(n, K + 1), u_draft=z(K, n), q=z(n * (K + 1), nh * hd),
        out=z(n * (K + 1), nh * hd)).items()}
    tables = hip.KvTables(page, n * cols, n, cols, b["table"].ptr, b["held"].ptr, b["refs"].ptr)

    def resize(lens):
        hip.check(L.syn_hip_kv_resize(C.byref(tables), R.dev(R.i32(lens)).ptr, b["ws"].ptr, 1 << 20, None))
        R.sync()

    def append(tokens, pos, seq):
        """keys and values (queries too: returned) of tokens at places of their sequences"""
        m = len(tokens)
        a = hip.KvAppend(layer=0, n_heads=nh, n_seqs=n, rotary_dim=0, interleaved=0, n_positions=most, eps=1e-6,
                         ldq=nh * hd, ldk=kv * hd, ldv=kv * hd, ldo=nh * hd, ld_table=cols)
        d = [R.dev(x[tokens]) for x in (eq, ek, ev)] + [R.dev(R.i32(x)) for x in (pos, seq)]
        q = hip.DeviceBuffer(m * nh * hd * 4)
        hip.check(L.syn_hip_kv_append(C.byref(pool.desc), C.byref(a), m, d[0].ptr, d[1].ptr, d[2].ptr, None, None,
                                      None, None, d[3].ptr, d[4].ptr, d[3].ptr, b["table"].ptr, q.ptr, None))
        R.sync()
        return q

    prompt = rng.integers(0, vocab, n_prompt)
    resize([n_prompt] + [0] * (n - 1))
    append(prompt, np.arange(n_prompt), np.zeros(n_prompt))
    lens = np.full(n, n_prompt)
    parent, dl = R.dev(R.i32(np.zeros(n))), R.dev(R.i32(lens))
    hip.check(L.syn_hip_kv_fork(C.byref(pool.desc), C.byref(tables), parent.ptr, dl.ptr, b["ws"].ptr, 1 << 20, None))
    R.sync()
    seqs = [list(prompt) for _ in range(n)]        # what the cache holds of each
    last, ended = rng.integers(0, vocab, n), np.zeros(n, bool)
    rejected = accepted = 0
    for step in range(rounds):
        ended[n - 1] = step >= 5                   # the last sample ends early
        room = np.where(ended, 0, lens + K + 1)
        resize(room)
        u, u_draft = rng.random((n, K + 1), f32), rng.random((K, n), f32)
        b["u"].upload(u), b["u_draft"].upload(u_draft)
        state = R.dev(R.i32(np.where(ended, -1, 0)))
        one = hip.DraftVerify(n_seqs=n, max_draft=0, pad=PAD, vocab=vocab, ld_target=ldl, target_stride=ldl)
        x, drafted, draft = last, np.zeros((n, K), np.int64), z(n, K, vocab)
        for i in range(K):
            rows = z(n, ldl)
            rows[:, :vocab] = draft[:, i] = draft_w[x]
            part = b["draft"].ptr + i * n * ldl * 4
            hip.check(L.syn_hip_memcpy_h2d(part, hip.ptr(rows), rows.nbytes))
            hip.check(L.syn_hip_draft_verify(C.byref(one), part, None, None, state.ptr, b["heat"].ptr,
                                             b["u_draft"].ptr + i * n * 4, b["x"].ptr, b["count"].ptr, None,
                                             b["ws"].ptr, 1 << 20, None))
            R.sync()
            x = b["x"].download((n,), np.int32).astype(np.int64)
            for s in range(n):
                want, m, _, near = D.verify(draft[s, i:i + 1], None, None, -1 if ended[s] else 0, heat[s],
                                            [u_draft[i, s]], PAD, 0)
                assert near > 2.0 ** -30 and x[s] == want[0], (step, i, s)
            drafted[:, i] = x
            x = np.minimum(x, vocab - 1)           # (an ended sample's pad)
        b["drafted"].upload(R.i32(drafted))
        ids = np.minimum(np.concatenate([last[:, None], drafted], 1), vocab - 1)
        pos = np.where(ended[:, None], -1, lens[:, None] + np.arange(K + 1))
        q = append(ids.reshape(-1), pos.reshape(-1), np.repeat(np.arange(n), K + 1))
        p = hip.PagedAttention(layer=0, n_heads=nh, n_seqs=n, n_tokens=n * (K + 1), max_new=K + 1, max_len=most,
                               window=0, scale=0.0, ldq=nh * hd, ldo=nh * hd, ld_table=cols)
        need = C.c_size_t()
        hip.check(L.syn_hip_paged_attention_workspace(C.byref(pool.desc), C.byref(p), C.byref(need)))
        assert need.value <= 1 << 20
        droom = R.dev(R.i32(room))
        hip.check(L.syn_hip_paged_attention(C.byref(pool.desc), C.byref(p), q.ptr, None, droom.ptr, b["table"].ptr,
                                            b["out"].ptr, b["ws"].ptr, 1 << 20, None))
        R.sync()
        out = b["out"].download((n, K + 1, nh * hd), f32)
        for s in np.flatnonzero(~ended):
            all_ = np.array(seqs[s] + ids[s].tolist())
            want, mag, qk = causal(eq[ids[s]].astype(np.float64).reshape(K + 1, nh, hd), stored["k"][all_],
                                   stored["v"][all_], lens[s] + np.arange(K + 1), 0, 1 / np.sqrt(hd))
            e = (hd + 8) * 2.0 ** -24 * qk[..., None] / np.sqrt(hd)
            tol = (2 * e + (len(all_) + 64) * 2.0 ** -24) * mag
            assert (np.abs(out[s].reshape(want.shape) - want) <= tol).all(), (step, s)
        logits = z(n, K + 1, ldl)
        logits[..., :vocab] = 0.15 * (out @ out_w) + draft_w[ids]
        b["logits"].upload(logits)
        n_draft = np.where(ended, -1, K)
        dn = R.dev(R.i32(n_draft))
        both = hip.DraftVerify(n_seqs=n, max_draft=K, pad=PAD, vocab=vocab, ld_target=ldl,
                               target_stride=(K + 1) * ldl, ld_draft=n * ldl, draft_stride=ldl)
        hip.check(L.syn_hip_draft_verify(C.byref(both), b["logits"].ptr, b["draft"].ptr, b["drafted"].ptr, dn.ptr,
                                         b["heat"].ptr, b["u"].ptr, b["tokens"].ptr, b["count"].ptr, None,
                                         b["ws"].ptr, 1 << 20, None))
        R.sync()
        tokens, count = b["tokens"].download((n, K + 1), np.int32), b["count"].download((n,), np.int32)
        for s in range(n):
            want, m, _, near = D.verify(logits[s, :, :vocab], draft[s], drafted[s], n_draft[s], heat[s], u[s],
                                        PAD, K)
            assert near > 2.0 ** -30 and count[s] == m and (tokens[s] == want).all(), (step, s)
            if ended[s]:
                continue
            rejected, accepted = rejected + (m <= K), accepted + (m > 1)
            seqs[s] += [last[s]] + tokens[s, :m - 1].tolist()
            last[s] = tokens[s, m - 1]
            lens[s] += m
            assert len(seqs[s]) == lens[s]
    assert rejected > 3 and accepted > 3
    refs, held = b["refs"].download((n * cols,), np.int32), b["held"].download((n,), np.int32)
    table = b["table"].download((n, cols), np.int32)
    assert held[n - 1] == 0 and (table[n - 1] == -1).all()
    assert (refs == np.bincount(table[table >= 0], minlength=n * cols)).all()
