"""The K-quant decoder and its beam search in float64, with the keys and values
that the beams attend to rounded to the pages' type, for the tests."""
import numpy as np

import oracle as O
import paged_ref as R
from synapse_amd import hip

TINY = dict(hidden=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, inter=512, vocab=301,
            max_seq=96, eps=1e-5, rope_theta=5e5)
FMTS = [hip.FMT_Q4_K] * 6 + [hip.FMT_Q6_K]


def shapes(cfg):
    h, qd, kvd = cfg["hidden"], cfg["n_heads"] * cfg["head_dim"], cfg["n_kv_heads"] * cfg["head_dim"]
    return [(qd, h), (kvd, h), (kvd, h), (h, qd), (cfg["inter"], h), (cfg["inter"], h), (h, cfg["inter"])]


def weights(cfg=TINY, seed=0x5EED0000, head_std=0.2):
    """embedding, block bytes of [layer][projection], and of the head"""
    emb = O.normal(cfg["vocab"] * cfg["hidden"], seed, 0.5).reshape(cfg["vocab"], cfg["hidden"])
    layers = [[hip.kquant_encode(f, O.normal(n * k, seed + 1 + 8 * layer + p, 0.06).reshape(n, k))
               for p, ((n, k), f) in enumerate(zip(shapes(cfg), FMTS))] for layer in range(cfg["n_layers"])]
    w = O.normal(cfg["vocab"] * cfg["hidden"], seed + 1 + 8 * cfg["n_layers"], head_std)
    return emb, layers, hip.kquant_encode(hip.FMT_Q6_K, w.reshape(cfg["vocab"], cfg["hidden"]))


def device_model(w, cfg=TINY, qk_norm=False):
    emb, layers, head = w
    g = hip.KQuantCausalLM(cfg, FMTS[0], FMTS[3], FMTS[4], FMTS[6], hip.FMT_Q6_K, qk_norm=qk_norm)
    g.set_embed(emb)
    for i, projs in enumerate(layers):
        for p, b in enumerate(projs):
            g.set_proj(i, p, b)
    g.set_lm_head(head)
    g.finalize()
    return g


class Model:
    def __init__(self, w, cfg=TINY, qk_norm=False, kv="f32"):
        self.c, self.qk_norm, self.kv = cfg, qk_norm, kv
        emb, layers, head = w
        self.emb = emb.astype(np.float64)
        self.w = [[hip.kquant_decode(f, b).astype(np.float64).reshape(n, k).T.copy()
                   for (n, k), f, b in zip(shapes(cfg), FMTS, projs)] for projs in layers]
        self.head = (hip.kquant_decode(hip.FMT_Q6_K, head).astype(np.float64)
                     .reshape(cfg["vocab"], cfg["hidden"]).T.copy())
        hd = cfg["head_dim"]
        i = np.arange(hd // 2, dtype=np.float32)
        freq = np.float32(1) / np.power(np.float32(cfg["rope_theta"]), np.float32(2) * i / np.float32(hd))
        ang = np.arange(cfg["max_seq"], dtype=np.float32)[:, None] * freq.astype(np.float32)
        self.cos, self.sin = np.cos(ang).astype(np.float64), np.sin(ang).astype(np.float64)

    def norm(self, x):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.c["eps"])

    def stored(self, x):
        return R.values(R.store(x.astype(np.float32), self.kv), self.kv) if self.kv != "f32" else x

    def qkv(self, layer, x, pos):
        c, hd = self.c, self.c["head_dim"]
        y = self.norm(x)
        q, k, v = ((y @ self.w[layer][p]).reshape(len(x), -1, hd) for p in range(3))
        if self.qk_norm:
            q, k = self.norm(q), self.norm(k)
        cos, sin = self.cos[pos][:, None], self.sin[pos][:, None]
        return R.rotate(q, cos, sin, hd, 0), R.rotate(k, cos, sin, hd, 0), v

    def rest(self, layer, x, attn):
        w = self.w[layer]
        x = x + attn.reshape(len(x), -1) @ w[3]
        y = self.norm(x)
        gate = y @ w[4]
        return x + (gate / (1 + np.exp(-gate)) * (y @ w[5])) @ w[6]

    def attend(self, q, k, v, mask):
        """q [n][heads][hd], k and v [n or 1][positions][kv heads][hd], mask [n][positions]"""
        rep = self.c["n_heads"] // self.c["n_kv_heads"]
        k, v = (np.repeat(np.broadcast_to(x, (len(q),) + x.shape[1:]), rep, 2) for x in (k, v))
        s = np.einsum("nhd,nphd->nhp", q, k) / np.sqrt(self.c["head_dim"])
        s = np.where(mask[:, None], s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        return np.einsum("nhp,nphd->nhd", p / p.sum(-1, keepdims=True), v)

    def prefill(self, ids):
        """logits of the last token; keys and values as stored, [layer][1][n][kv heads][hd]"""
        n = len(ids)
        x, ks, vs = self.emb[ids], [], []
        for layer in range(self.c["n_layers"]):
            q, k, v = self.qkv(layer, x, np.arange(n))
            x = self.rest(layer, x, self.attend(q, k[None], v[None], np.tril(np.ones((n, n), bool))))
            ks.append(self.stored(k)[None])
            vs.append(self.stored(v)[None])
        return (self.norm(x[-1:]) @ self.head)[0], ks, vs

    def step(self, tokens, pos, ks, vs):
        """one token of every row: logits, and keys and values with it"""
        x, nk, nv = self.emb[tokens], [], []
        for layer in range(self.c["n_layers"]):
            q, k, v = self.qkv(layer, x, np.full(len(tokens), pos))
            k = np.concatenate([ks[layer], self.stored(k)[:, None]], 1)
            v = np.concatenate([vs[layer], self.stored(v)[:, None]], 1)
            x = self.rest(layer, x, self.attend(q, k, v, np.ones(k.shape[:2], bool)))
            nk.append(k)
            nv.append(v)
        return self.norm(x) @ self.head, nk, nv


def logp(x):
    d = x - x.max(-1, keepdims=True)
    return d - np.log(np.exp(d).sum(-1, keepdims=True))


def search(model, prompt, max_new, W, eos):
    """The beams as {tokens up to the eos: score}; the least distance, over all
    choices, between the last continuation that was taken and the first that was
    not; how many beams had ended before the last token."""
    logits, ks, vs = model.prefill(prompt)
    val = logp(logits)[None]
    first, gap, early = True, np.inf, 0
    for step in range(max_new):
        v = val.shape[1]
        order = np.argsort(-val.reshape(-1), kind="stable")[:W + 1]
        best = val.reshape(-1)[order]
        if len(order) > W and np.isfinite(best[W]):
            gap = min(gap, best[W - 1] - best[W])
        parent, token = np.divmod(order[:W], v)
        scores = best[:W]
        if first:
            beams, done = [[int(t)] for t in token], token == eos
            ks, vs = ([np.repeat(x, W, 0) for x in y] for y in (ks, vs))
            first = False
        else:
            beams = [beams[p] + ([] if done[p] else [int(t)]) for p, t in zip(parent, token)]
            ks, vs = ([x[parent] for x in y] for y in (ks, vs))
            done = done[parent] | (token == eos)
        if step == max_new - 1:
            break
        early = int(done.sum())
        logits, ks, vs = model.step(token, len(prompt) + step, ks, vs)
        only = np.full(v, -np.inf)
        only[max(eos, 0)] = 0.0
        val = np.where(done[:, None], only, logp(logits)) + scores[:, None]
    return {tuple(b): float(s) for b, s in zip(beams, scores)}, gap, early


# How far a score of the device may be from the definition's, and half of the gap
# that the choices of a case have (test_klm_search_ref.py holds them to it):
# - every product sums at most 512 terms in f32 (3e-5 of the terms' sum, logits up
#   to ten, twenty tokens): 1e-3;
# - a key or value of 16 bits lies one step (2^-10 of itself in f16, 2^-7 in bf16)
#   from the definition's where the two f32 sums are on both sides of a rounding: one
#   of some 15000 moves a score by 2^-7 / 8 of one term of a dot product, and few
#   do: 1e-2;
# - more than 8 rows (of beams, or of the prompt) have their products' operands
#   rounded to f16 once, 2^-11 each: logits of ten off by 5e-3, several tokens: 2e-2.
F32, PAGES, ROWS = 1e-3, 1e-2, 2e-2
# beams, prompt length, new tokens, pages, head norms, prompt's seed, eos, bound
CASES = [(4, 8, 20, "f32", False, 0, -1, F32), (4, 8, 20, "f32", False, 1, 219, F32),
         (8, 5, 20, "f32", True, 0, -1, F32), (8, 5, 20, "f32", True, 0, 139, F32),
         (4, 8, 20, "f16", True, 0, -1, PAGES), (4, 8, 20, "f16", True, 40, 252, PAGES),
         (8, 7, 18, "bf16", False, 2, -1, PAGES), (8, 7, 18, "bf16", False, 82, 60, PAGES),
         (2, 1, 40, "f16", False, 40, -1, PAGES), (2, 1, 40, "f16", False, 1, 135, PAGES),
         (2, 1, 40, "f16", False, 1, 280, PAGES),  # all beams end, and the search with them
         (7, 1, 17, "bf16", True, 34, -1, PAGES), (7, 1, 17, "bf16", True, 5, 99, PAGES),
         (12, 33, 6, "f32", True, 33, -1, ROWS), (12, 33, 6, "f32", True, 33, 75, ROWS),
         (4, 21, 12, "f16", False, 4, -1, ROWS), (4, 21, 12, "f16", False, 2, 167, ROWS),
         (16, 40, 4, "bf16", False, 13, -1, ROWS), (64, 9, 3, "f16", True, 653, -1, ROWS)]


def prompt_of(case):
    return O.token_ids(case[1], 0x5EED0000 + case[5], TINY["vocab"])
