"""Beam search with the K-quant decoder, against a search in float64 over the
oracle's logits, and the operators of a step run together by hand.

The decoder's logits differ from the oracle's by the float tolerance of its
path; DELTA bounds that for these models (logits of a few units, per-step
relative differences below 1e-3 in test_gpu_klm.py), and a search is compared
token by token as long as no choice in it was closer than that."""
import ctypes as C

import numpy as np
import pytest

import oracle as O
import paged_ref as R
from synapse_amd import hip

pytestmark = pytest.mark.gpu
DELTA = 2e-2


@pytest.fixture(scope="module", autouse=True)
def gpu():
    hip.init(0)


TINY = dict(hidden=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, inter=512, vocab=301,
            max_seq=96, eps=1e-5, rope_theta=5e5)


def build(cfg=TINY, qk_norm=False, seed=0x5EED0000, head_std=0.2):
    o = O.CausalLM(cfg, qk_norm=qk_norm)
    f4, f6 = hip.FMT_Q4_K, hip.FMT_Q6_K
    g = hip.KQuantCausalLM(cfg, f4, f4, f4, f6, f6, qk_norm=qk_norm)
    h, qd = cfg["hidden"], cfg["n_heads"] * cfg["head_dim"]
    kvd, inter = cfg["n_kv_heads"] * cfg["head_dim"], cfg["inter"]
    emb = O.normal(cfg["vocab"] * h, seed, 0.5).reshape(cfg["vocab"], h)
    o.set_embed(emb)
    g.set_embed(emb)
    shapes = [(qd, h, f4), (kvd, h, f4), (kvd, h, f4), (h, qd, f4), (inter, h, f4), (inter, h, f4),
              (h, inter, f6)]
    names = {f4: "q4_k", f6: "q6_k"}
    for layer in range(cfg["n_layers"]):
        for p, (n, k, f) in enumerate(shapes):
            b = hip.kquant_encode(f, O.normal(n * k, seed + 1 + 8 * layer + p, 0.06).reshape(n, k))
            o.set_proj(layer, p, names[f], b)
            g.set_proj(layer, p, b)
    w = O.normal(cfg["vocab"] * h, seed + 1 + 8 * cfg["n_layers"], head_std).reshape(cfg["vocab"], h)
    b = hip.kquant_encode(f6, w)
    o.set_lm_head("q6_k", b)
    g.set_lm_head(b)
    g.finalize()
    return o, g


def logp(x):
    x = x.astype(np.float64)
    return x - x.max() - np.log(np.exp(x - x.max()).sum())


def search(o, prompt, max_new, W, eos):
    """beams as (score, tokens, finished), best first at every step, and the closest choice"""
    close = np.inf
    lp = logp(o.prefill(prompt))
    order = np.argsort(-lp, kind="stable")
    close = min(close, lp[order[W - 1]] - lp[order[W]], np.diff(-lp[order[:W]]).min() if W > 1 else np.inf)
    beams = [(lp[t], [int(t)], int(t) == eos) for t in order[:W]]
    for _ in range(max_new - 1):
        cand = []
        for b, (s, toks, fin) in enumerate(beams):
            if fin:
                cand.append((s, b, eos))
                continue
            x = logp(o.prefill(np.concatenate([prompt, np.uint32(toks)])))
            cand += [(s + x[t], b, int(t)) for t in np.argsort(-x, kind="stable")[:W + 1]]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        close = min([close] + [cand[i][0] - cand[i + 1][0] for i in range(min(W, len(cand) - 1))])
        beams = [(s, beams[b][1] + [t], beams[b][2] or t == eos) for s, b, t in cand[:W]]
    return beams, close


@pytest.mark.parametrize("W,plen,max_new,kv,qk_norm,graph", [
    (1, 9, 12, hip.KV_F32, False, True), (4, 21, 20, hip.KV_F32, False, True),
    (4, 21, 20, hip.KV_F32, False, False), (3, 1, 18, hip.KV_F16, True, True),
    (8, 40, 10, hip.KV_BF16, False, True), (12, 33, 6, hip.KV_F32, True, True),
    (5, 16, 1, hip.KV_F32, False, True), (2, 17, 34, hip.KV_F16, False, True)])
@pytest.mark.parametrize("eos", [-1, 7])
def test_beam_search(W, plen, max_new, kv, qk_norm, graph, eos):
    o, g = build(qk_norm=qk_norm)
    g.set_options(True, graph)
    prompt = O.token_ids(plen, 0x5EED0000 + 77 + plen, TINY["vocab"])
    toks, lens, scores = g.generate_beams(prompt, max_new, W, eos, kv)
    assert (np.diff(scores) <= 0).all()
    for r in range(W):  # every beam's score is that of its tokens
        t = toks[r, :lens[r]]
        assert lens[r] == max_new or t[-1] == eos
        assert (toks[r, lens[r]:] == eos).all() and (eos not in t[:-1].tolist() or eos < 0)
        want, ids = 0.0, prompt
        for x in t:
            want += logp(o.prefill(ids))[x]
            ids = np.concatenate([ids, [x]]).astype(np.uint32)
        assert abs(want - scores[r]) <= DELTA, (r, want, scores[r])
    beams, close = search(o, prompt, max_new, W, eos)
    print("closest choice", close)
    assert abs(max(b[0] for b in beams) - scores[0]) <= DELTA or close < 2 * DELTA
    if close >= 2 * DELTA:
        for r, (s, t, fin) in enumerate(sorted(beams, key=lambda b: -b[0])):
            n = t.index(eos) + 1 if fin else len(t)
            assert toks[r, :lens[r]].tolist() == t[:n]


def test_one_beam_is_greedy_and_calls_repeat():
    _, g = build()
    prompt = O.token_ids(30, 5, TINY["vocab"])
    toks, _, s1 = g.generate_beams(prompt, 24, 1)
    greedy, margins = g.generate(prompt, 24)
    n = 24 if (margins > DELTA).all() else int(np.argmin(margins > DELTA))
    assert n >= 3 and toks[0, :n].tolist() == greedy[:n].tolist()
    a = g.generate_beams(prompt, 20, 6)
    b = g.generate_beams(prompt, 20, 6)          # the same graph again
    c = g.generate_beams(prompt[:11], 9, 4, eos=3)  # another shape between
    d = g.generate_beams(prompt, 20, 6)
    for x, y in ((a, b), (a, d)):
        assert all(np.array_equal(p, q) for p, q in zip(x, y))
    assert c[0].shape == (4, 9)
    g.set_options(True, False)
    assert all(np.array_equal(p, q) for p, q in zip(a, g.generate_beams(prompt, 20, 6)))
    # the model's own cache holds the prompt
    assert g.cache_len() == 30
    assert g.generate(prompt, 24)[0].tolist() == greedy.tolist()


def test_length_penalty_orders_the_beams():
    _, g = build()
    prompt = O.token_ids(12, 9, TINY["vocab"])
    toks, lens, scores = g.generate_beams(prompt, 15, 5)
    eos = int(toks[1, 4])
    for alpha in (0.0, 1.0, 2.0):
        t, n, s = g.generate_beams(prompt, 15, 5, eos=eos, length_penalty=alpha)
        rank = s / n.astype(np.float64) ** alpha
        assert (np.diff(rank) <= 1e-12).all()


def test_extreme_length_penalties_keep_an_order():
    _, g = build()
    prompt = O.token_ids(12, 9, TINY["vocab"])
    plain = g.generate_beams(prompt, 15, 5, eos=3)
    for alpha in (-3e38, 3e38):
        toks, lens, scores = g.generate_beams(prompt, 15, 5, eos=3, length_penalty=alpha)
        assert sorted(scores.tolist()) == sorted(plain[2].tolist())


def test_weights_set_again_between_searches():
    """the captured step does not outlive the buffers that it reads"""
    _, g = build()
    _, want = build(head_std=0.3)
    prompt = O.token_ids(20, 4, TINY["vocab"])
    g.generate_beams(prompt, 9, 4)
    n = TINY["vocab"] * TINY["hidden"]
    w = O.normal(n, 0x5EED0000 + 1 + 8 * TINY["n_layers"], 0.3).reshape(TINY["vocab"], TINY["hidden"])
    g.set_lm_head(hip.kquant_encode(hip.FMT_Q6_K, w))
    g.finalize()
    for a, b in zip(g.generate_beams(prompt, 9, 4), want.generate_beams(prompt, 9, 4)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("kw", [dict(n_beams=0), dict(n_beams=65), dict(eos=301), dict(kv_dtype=3),
                                dict(max_new=90), dict(plen=0), dict(plen=97),
                                dict(penalty=float("nan")), dict(penalty=float("inf"))])
def test_refusals(kw):
    _, g = build()
    d = dict(n_beams=4, eos=-1, kv_dtype=0, max_new=8, plen=10, penalty=0.0)
    d.update(kw)
    prompt = np.zeros(max(d["plen"], 1), np.uint32)
    p = hip.BeamSearch(d["n_beams"], d["eos"], d["kv_dtype"], d["penalty"])
    out = np.zeros((65, 96), np.uint32)
    assert hip.lib().syn_hip_klm_generate_beams(g.h, hip.ptr(prompt), d["plen"], d["max_new"],
                                                C.byref(p), hip.ptr(out), None, None) == 2


# ---------------------------------------------------------------- the operators together
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_steps_by_hand(dtype):
    """Two groups of four beams over one attention layer: append, attend,
    choose, reorder, for enough steps to cross pages; the host keeps every
    beam's own list of rows."""
    rng = np.random.default_rng(3)
    G, W, nh, kv, hd, ps, V, steps = 2, 4, 4, 2, 64, 8, 500, 21
    rows, plen, cols = G * W, [19, 8], 3
    n_pages = 3 + 1 + rows * (cols + 1)
    pool = R.Pool(dtype, ps, n_pages, 1, kv, hd, fill=float("nan"))
    ids = R.i32(np.arange(n_pages))
    ptable = R.i32([[0, 1, 2], [3, -1, -1]])
    table = R.i32(ids[4:4 + rows * cols].reshape(rows, cols))
    spare = R.i32(ids[4 + rows * cols:])
    ang = rng.uniform(-3, 3, (64, hd // 2)).astype(np.float32)
    cos, sin = np.cos(ang), np.sin(ang)
    ld = (nh + 2 * kv) * hd
    L = hip.lib()
    dev = {k: R.dev(v) for k, v in dict(ptable=ptable, table=table, spare=spare, cos=cos, sin=sin,
                                        plen=R.i32(plen)).items()}

    def append(x, pos, seq, index, tab, n_seqs, ldt, out):
        p = hip.KvAppend(layer=0, n_heads=nh, n_seqs=n_seqs, rotary_dim=hd, interleaved=0, n_positions=64,
                         eps=0, ldq=ld, ldk=ld, ldv=ld, ldo=nh * hd, ld_table=ldt)
        b = [R.dev(x), R.dev(R.i32(pos)), R.dev(R.i32(seq)), R.dev(R.i32(index))]
        hip.check(L.syn_hip_kv_append(C.byref(pool.desc), C.byref(p), len(x), b[0].ptr,
                                      b[0].ptr + 4 * nh * hd, b[0].ptr + 4 * (nh + kv) * hd, None, None,
                                      dev["cos"].ptr, dev["sin"].ptr, b[1].ptr, b[2].ptr, b[3].ptr,
                                      tab.ptr, out.ptr, None))
        R.sync()

    def stored(x, pos):
        """what a token leaves in the cache"""
        y = x.astype(np.float64).reshape(nh + 2 * kv, hd)
        k = R.rotate(y[nh:nh + kv], cos[pos].astype(np.float64), sin[pos].astype(np.float64), hd, 0)
        return (R.values(R.store(k.astype(np.float32), dtype), dtype),
                R.values(R.store(y[nh + kv:].astype(np.float32), dtype), dtype))

    prefix = []
    for g in range(G):
        x = rng.standard_normal((plen[g], ld)).astype(np.float32)
        append(x, range(plen[g]), [g] * plen[g], range(plen[g]), dev["ptable"], G, 3,
               R.dev(np.zeros((plen[g], nh * hd), np.float32)))
        prefix.append([stored(x[i], i) for i in range(plen[g])])
    ap = hip.PrefixAttention(layer=0, n_heads=nh, n_groups=G, group_size=W, max_prefix=19,
                             max_suffix=steps, scale=0.0, ldq=nh * hd, ldo=nh * hd, ld_prefix_table=3,
                             ld_table=cols)
    sp = hip.BeamSelect(n_groups=G, n_beams=W, n_select=W, eos=-1, pad=0, vocab=V, ld_logits=V)
    need = C.c_size_t()
    hip.check(L.syn_hip_prefix_attention_workspace(C.byref(pool.desc), C.byref(ap), C.byref(need)))
    aws, an = hip.DeviceBuffer(need.value), need.value
    hip.check(L.syn_hip_beam_select_workspace(C.byref(sp), C.byref(need)))
    sws, sn = hip.DeviceBuffer(need.value), need.value
    q, out = hip.DeviceBuffer(rows * nh * hd * 4), hip.DeviceBuffer(rows * nh * hd * 4)
    parent, token = hip.DeviceBuffer(rows * 4), hip.DeviceBuffer(rows * 4)
    scores = rng.standard_normal(rows).astype(np.float32)
    ds = R.dev(scores)
    mine = [[] for _ in range(rows)]
    for step in range(steps):
        x = rng.standard_normal((rows, ld)).astype(np.float32)
        pos = [plen[r // W] + step for r in range(rows)]
        append(x, pos, range(rows), [step] * rows, dev["table"], rows, cols, q)
        for r in range(rows):
            mine[r] = mine[r] + [stored(x[r], pos[r])]
        dl = R.dev(R.i32([step + 1] * rows))
        hip.check(L.syn_hip_prefix_attention(C.byref(pool.desc), C.byref(ap), q.ptr, dev["ptable"].ptr,
                                             dev["plen"].ptr, dev["table"].ptr, dl.ptr, out.ptr, aws.ptr,
                                             an, None))
        R.sync()
        got = out.download((rows, nh, hd), np.float32)
        turned = q.download((rows, nh, hd), np.float32).astype(np.float64)
        for r in range(rows):
            kvs = prefix[r // W] + mine[r]
            k, v = np.stack([a for a, _ in kvs]), np.stack([b for _, b in kvs])
            want, mag, qk = R.attention(turned[r], k, v, 1 / 8)
            # keys and values may be one step of their type off the definition's where it lies between two
            step_of = 0 if dtype == "f32" else 2 * R.HALF_STEP[dtype]
            e = ((hd + 8) * 2.0 ** -24 + step_of) * qk / 8 + 12 * 2.0 ** -24 * qk / 8
            assert (np.abs(got[r] - want) <= (2 * e + (len(k) + 64) * 2.0 ** -24 + step_of) * mag).all(), step
        logits = (rng.standard_normal((rows, V)) * 2).astype(np.float32)
        dx = R.dev(logits)
        hip.check(L.syn_hip_beam_select(C.byref(sp), dx.ptr, ds.ptr, None, parent.ptr, token.ptr, ds.ptr,
                                        None, sws.ptr, sn, None))
        held = R.dev(R.i32([step + 1] * G))
        hip.check(L.syn_hip_beam_reorder_pages(C.byref(pool.desc), G, W, parent.ptr, held.ptr,
                                               dev["table"].ptr, cols, dev["spare"].ptr, None))
        R.sync()
        par = parent.download((rows,), np.int32)
        new = ds.download((rows,), np.float32)
        for g in range(G):
            s = slice(g * W, (g + 1) * W)
            p, t, v, _ = R.select(logits[s], scores[s].astype(np.float64), np.zeros(W), W, -1, 0)
            assert np.array_equal(par[s], p)
            assert np.array_equal(token.download((rows,), np.int32)[s], t)
        scores = new
        mine = [mine[r // W * W + par[r]] for r in range(rows)]


@pytest.mark.parametrize("W,plen,max_new,eos", [(4, 21, 20, -1), (3, 1, 18, 7), (6, 40, 12, -1), (2, 17, 30, 11)])
def test_beam_search_over_the_decoders_own_logits(W, plen, max_new, eos):
    """The same prefill, and the decoder's own single steps: both sides sum in
    f32 in different orders (512 terms: 3e-5 relative, logits up to about ten),
    so choices more than 1e-3 apart are the same."""
    _, g = build()

    class Own:
        def prefill(self, ids):
            lg = g.prefill(ids[:plen])
            for t in ids[plen:]:
                lg = g.forward_one(int(t))
            return lg

    prompt = O.token_ids(plen, 0x5EED0000 + 77 + plen, TINY["vocab"])
    beams, close = search(Own(), prompt, max_new, W, eos)
    toks, lens, scores = g.generate_beams(prompt, max_new, W, eos)
    best = sorted(beams, key=lambda b: -b[0])
    assert abs(best[0][0] - scores[0]) <= 1e-3 or close < 2e-3
    if close >= 2e-3:
        for r, (s, t, fin) in enumerate(best):
            n = t.index(eos) + 1 if fin else len(t)
            assert toks[r, :lens[r]].tolist() == t[:n] and abs(s - scores[r]) <= 1e-3
