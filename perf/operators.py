"""Decoding several continuations of a prompt together: the operators, as cases to be timed.

- ``append``: keys and values of a batch of tokens into a paged cache, head
  norms and position rotation on the way (``syn_hip_kv_append``).
- ``attend``: one query token per sequence over a prefix that the sequences of
  a group share and a suffix of their own (``syn_hip_prefix_attention``).
- ``select``: the best continuations over beams and vocabulary
  (``syn_hip_beam_select``).
- ``rows``, ``pages``: states that follow the chosen beams
  (``syn_hip_beam_reorder_rows``, ``syn_hip_beam_reorder_pages``).

A page holds ``page`` positions of one layer's keys as [kv head][dim / 8][position][8]
and values as [kv head][position / 8][dim][8].
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KV_CODE = {"f32": 0, "f16": 1, "bf16": 2}
# (query heads, kv heads, head size) of the decoders' attention layers:
# Qwen3-0.6B, LLaMA-3.2-3B, LLaMA-3.2-1B and LFM2.5-350M, Mistral-7B
HEADS = {"qwen": (16, 8, 128), "llama3b": (24, 8, 128), "llama1b": (32, 8, 64),
         "lfm": (16, 8, 64), "mistral": (32, 8, 128)}
VOCABS = (32000, 65536, 128256, 151936)


def listed():
    return [
        # one decode step of 8 beams: launch latency
        dict(name="append_step", kind="append", heads="llama3b", dtype="f32", tokens=8, seqs=8,
             start=40, page=16, norm=False, pad=0),
        # prompts of several requests, packed and padded, with q/k head norms
        dict(name="append_batch", kind="append", heads="qwen", dtype="bf16", tokens=517, seqs=5,
             start=0, page=64, norm=True, pad=11),
        # one long prompt
        dict(name="append_prompt", kind="append", heads="mistral", dtype="f16", tokens=8192,
             seqs=1, start=0, page=64, norm=False, pad=0),
        # four beams of a short prompt, early in the answer: latency
        dict(name="attend_short", kind="attend", heads="qwen", dtype="f32", groups=1, members=4,
             prefix=96, suffix=17, page=16),
        # eight beams of a document
        dict(name="attend_beams", kind="attend", heads="llama3b", dtype="f16", groups=1, members=8,
             prefix=4001, suffix=120, page=16),
        # requests that share a system prompt, each with a conversation of its own
        dict(name="attend_requests", kind="attend", heads="llama1b", dtype="bf16", groups=1,
             members=48, prefix=8200, suffix=1500, page=64),
        # four long documents, sixteen continuations each
        dict(name="attend_long", kind="attend", heads="mistral", dtype="f16", groups=4, members=16,
             prefix=32768, suffix=300, page=64),
        # four beams over a small vocabulary: latency
        dict(name="select_small", kind="select", groups=1, beams=4, select=4, vocab=32000, done=0),
        # four requests of eight beams, some finished
        dict(name="select_batch", kind="select", groups=4, beams=8, select=8, vocab=128256, done=3),
        # sixteen requests, twice the beams kept for the caller to filter
        dict(name="select_large", kind="select", groups=16, beams=8, select=16, vocab=151936,
             done=0),
        # the recurrent states of 48 Mamba-370M layers, eight beams
        dict(name="reorder_states", kind="rows", groups=1, beams=8, buffers=48, row=2048 * 16 * 4),
        # the paged cache of LLaMA-3.2-3B, four requests of eight beams
        dict(name="reorder_pages", kind="pages", heads="llama3b", dtype="f16", layers=28, groups=4,
             beams=8, held=171, room=256, page=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("append", "attend", "select", "rows", "pages"), (5, 7, 5, 2, 3))[0]
    heads, dtype = rng.choice(sorted(HEADS)), rng.choice(sorted(DTYPE))
    page = rng.choice((8, 16, 32, 64, 128))
    if kind == "append":
        tokens = _log_int(rng, 1, 8192)
        return dict(kind=kind, heads=heads, dtype=dtype, tokens=tokens,
                    seqs=rng.randrange(1, min(tokens, 64) + 1), start=rng.randrange(0, 300),
                    page=page, norm=rng.random() < 0.5, pad=min(tokens - 1, rng.randrange(0, 12)))
    if kind == "attend":
        groups, members = _log_int(rng, 1, 8), _log_int(rng, 1, 64)
        c = dict(kind=kind, heads=heads, dtype=dtype, groups=groups, members=members,
                 prefix=_log_int(rng, 16, 32768),
                 suffix=_log_int(rng, 1, max(2, min(2048, 65536 // (groups * members)))), page=page)
        while work(c)["bytes"] > 4e8 or work(c)["flops"] > 2e10:
            c["prefix"], c["suffix"] = c["prefix"] * 3 // 4, max(1, c["suffix"] * 3 // 4)
        return c
    if kind == "select":
        beams = rng.randrange(1, 17)
        vocab = rng.choice(VOCABS) - (rng.randrange(1, 64) if rng.random() < 0.5 else 0)
        return dict(kind=kind, groups=_log_int(rng, 1, max(1, 128 // beams)), beams=beams,
                    select=beams * rng.choice((1, 1, 2)), vocab=vocab,
                    done=rng.randrange(0, beams))
    beams = rng.randrange(2, 17)
    if kind == "rows":
        row = 4 * _log_int(rng, 16, 2048 * 16)
        return dict(kind=kind, groups=rng.randrange(1, 5), beams=beams,
                    buffers=max(1, min(rng.randrange(1, 49), 48 * 8 // (4 * beams))), row=row)
    room = page * rng.randrange(2, 1 + max(2, 512 // page))
    return dict(kind=kind, heads=heads, dtype=dtype, layers=rng.randrange(1, 17),
                groups=rng.randrange(1, 3), beams=beams, held=rng.randrange(1, room), room=room,
                page=page)


# ---------------------------------------------------------------- prepare
def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000 + salt)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ints(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)


def _pool(g, c, layers, pages):
    """a pool of keys and one of values, every place filled"""
    _, kv, hd = HEADS[c["heads"]]
    k = torch.empty((layers, pages, kv, hd // 8, c["page"], 8), device="cuda", dtype=DTYPE[c["dtype"]])
    v = torch.empty((layers, pages, kv, c["page"] // 8, hd, 8), device="cuda", dtype=DTYPE[c["dtype"]])
    k.normal_(generator=g)
    v.normal_(generator=g)
    return k, v


def _pages(g, n, *shape):
    """a table of distinct pages, in no order"""
    return torch.randperm(n, generator=g, device="cuda")[:math.prod(shape)].int().reshape(shape)


def _up(a, b):
    return -(-a // b)


def _prepare_append(c, seed):
    g = _gen(seed)
    nh, kv, hd = HEADS[c["heads"]]
    t, pad, n = c["tokens"], c["pad"], c["seqs"]
    # the packed rows of the sequences' new tokens, of about equal number, then padding
    seq = (torch.arange(t - pad, device="cuda") * n // (t - pad)).int()
    first = torch.searchsorted(seq, torch.arange(n, device="cuda", dtype=torch.int32))
    index = torch.arange(t - pad, device="cuda") - first[seq.long()] + c["start"]
    fill = torch.zeros(pad, device="cuda", dtype=torch.int32)
    index = torch.cat([index.int(), fill - 1])
    cols = _up(c["start"] + _up(t - pad, n) + 1, c["page"])
    k, v = _pool(g, c, 1, n * cols)
    positions = cols * c["page"]
    freq = 1e6 ** (-torch.arange(hd // 2, device="cuda", dtype=torch.float64) * 2 / hd)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    return dict(c, k=k, v=v, qkv=_randn(g, t, (nh + 2 * kv) * hd), seq=torch.cat([seq, fill]),
                index=index, pos=index.clamp(min=0), table=_pages(g, n * cols, n, cols),
                cos=angle.cos().float(), sin=angle.sin().float(),
                qn=1 + 0.1 * _randn(g, hd) if c["norm"] else None,
                kn=1 + 0.1 * _randn(g, hd) if c["norm"] else None,
                out=torch.zeros((t, nh * hd), device="cuda"))


def _prepare_attend(c, seed):
    g = _gen(seed)
    nh, kv, hd = HEADS[c["heads"]]
    rows = c["groups"] * c["members"]
    pc, sc = _up(c["prefix"], c["page"]), _up(c["suffix"], c["page"])
    n = c["groups"] * pc + rows * sc
    k, v = _pool(g, c, 1, n)
    table = _pages(g, n, n)
    # the longest prefix and the longest suffix are the case's; others are up to half shorter
    plen = c["prefix"] - _ints(g, 0, c["prefix"] // 2 + 1, c["groups"])
    slen = c["suffix"] - _ints(g, 0, c["suffix"] // 2 + 1, rows)
    plen[0], slen[rows // 2] = c["prefix"], c["suffix"]
    return dict(c, k=k, v=v, q=_randn(g, rows, nh * hd), out=torch.zeros((rows, nh * hd), device="cuda"),
                ptable=table[:c["groups"] * pc].reshape(c["groups"], pc).contiguous(), plen=plen,
                table=table[c["groups"] * pc:].reshape(rows, sc).contiguous(), slen=slen,
                # scratch of the split attention: as much as any split of this work may ask for
                scratch=torch.empty(256 << 20, device="cuda", dtype=torch.uint8))


def _prepare_select(c, seed):
    g = _gen(seed)
    rows = c["groups"] * c["beams"]
    logits = _randn(g, rows, c["vocab"]) * 2.5
    logits[:, :: 1009] = -math.inf  # words that the caller bans
    done = torch.zeros((c["groups"], c["beams"]), device="cuda", dtype=torch.int32)
    done[:, c["beams"] - c["done"]:] = 1
    scores = -torch.rand(rows, generator=g, device="cuda") * 3 - 20
    picked = c["groups"] * c["select"]
    return dict(c, logits=logits, finished=done.reshape(-1), scores=scores,
                eos=2, parent=torch.zeros(picked, device="cuda", dtype=torch.int32),
                token=torch.zeros(picked, device="cuda", dtype=torch.int32),
                score=torch.zeros(picked, device="cuda"),
                ended=torch.zeros(picked, device="cuda", dtype=torch.int32),
                scratch=torch.empty(16 << 20, device="cuda", dtype=torch.uint8))


def _parents(g, groups, beams):
    """the better half of the beams stays where it is, the others follow one of them"""
    keep = _up(beams, 2)
    parent = torch.arange(beams, device="cuda", dtype=torch.int32).repeat(groups, 1)
    parent[:, keep:] = _ints(g, 0, keep, groups, beams - keep)
    return parent.reshape(-1)


def _prepare_rows(c, seed):
    g = _gen(seed)
    return dict(c, parent=_parents(g, c["groups"], c["beams"]),
                rows=_randn(g, c["buffers"], c["groups"] * c["beams"], c["row"] // 4))


def _prepare_pages(c, seed):
    g = _gen(seed)
    rows, cols = c["groups"] * c["beams"], c["room"] // c["page"]
    k, v = _pool(g, c, c["layers"], rows * (cols + 1))
    held = c["held"] - _ints(g, 0, min(c["held"], c["page"] // 2), c["groups"])
    held[0] = c["held"]
    ids = _pages(g, rows * (cols + 1), rows * (cols + 1))
    return dict(c, k=k, v=v, len=held, parent=_parents(g, c["groups"], c["beams"]),
                table=ids[:rows * cols].reshape(rows, cols).contiguous(),
                spare=ids[rows * cols:].contiguous())


def prepare(case, seed):
    return {"append": _prepare_append, "attend": _prepare_attend, "select": _prepare_select,
            "rows": _prepare_rows, "pages": _prepare_pages}[case["kind"]](dict(case), seed)


# ---------------------------------------------------------------- run, plain
def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _norm(x, gain):
    return x if gain is None else x * gain * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)


def _plain_append(s):
    nh, kv, hd = HEADS[s["heads"]]
    t = s["tokens"]
    q, k, v = s["qkv"].reshape(t, nh + 2 * kv, hd).split((nh, kv, kv), 1)
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    s["out"].copy_(_rotate(_norm(q, s["qn"]), cos, sin).reshape(t, -1))
    k = _rotate(_norm(k, s["kn"]), cos, sin)
    n = t - s["pad"]  # the padding rows come last
    index = s["index"][:n].long()
    page, slot = s["table"][s["seq"][:n].long(), index // s["page"]].long(), index % s["page"]
    s["k"][0][page, :, :, slot] = k[:n].reshape(n, kv, hd // 8, 8).to(s["k"].dtype)
    s["v"][0].permute(0, 2, 4, 1, 3)[page, slot // 8, slot % 8] = v[:n].to(s["v"].dtype)
    return [s["out"], s["k"], s["v"]]


def _keys(s, table):
    """[table rows, kv head, position, dim] in float32"""
    x = s["k"][0][table.long()].float()  # rows, pages, kv, dim / 8, position, 8
    return x.permute(0, 2, 1, 4, 3, 5).flatten(4, 5).flatten(2, 3)


def _values(s, table):
    x = s["v"][0][table.long()].float()  # rows, pages, kv, position / 8, dim, 8
    return x.permute(0, 2, 1, 3, 5, 4).flatten(2, 4)


def _scores(q, k, length, scale):
    s = (q @ k.transpose(-1, -2).contiguous()) * scale
    off = torch.arange(k.shape[-2], device="cuda") >= length[:, None]
    return s.masked_fill(off[:, None, None], -math.inf)


def _plain_attend(s):
    nh, kv, hd = HEADS[s["heads"]]
    g, m, rep, scale = s["groups"], s["members"], nh // kv, 1 / math.sqrt(hd)
    q = s["q"].reshape(g, m, kv, rep, hd).transpose(1, 2)  # group, kv, member, rep, dim
    a = _scores(q.reshape(g, kv, m * rep, hd), _keys(s, s["ptable"]), s["plen"], scale)
    mine = s["q"].reshape(g * m, kv, rep, hd)
    b = _scores(mine, _keys(s, s["table"]), s["slen"], scale)
    per = lambda x: x.reshape(g, kv, m, rep, -1).transpose(1, 2).reshape(g * m, kv, rep, -1)
    back = lambda x: x.reshape(g, m, kv, rep, -1).transpose(1, 2).reshape(g, kv, m * rep, -1)
    top = torch.maximum(per(a.amax(-1, keepdim=True)), b.amax(-1, keepdim=True))
    a, b = torch.exp(a - back(top)), torch.exp(b - top)
    total = per(a.sum(-1, keepdim=True)) + b.sum(-1, keepdim=True)
    out = (per(a @ _values(s, s["ptable"])) + b @ _values(s, s["table"])) / total
    return out.reshape(g * m, nh * hd)


def _plain_select(s):
    g, w, v = s["groups"], s["beams"], s["vocab"]
    x = s["logits"].double()  # two candidates may lie closer than 32 bits tell
    x = x - (x - x.amax(-1, keepdim=True)).exp().sum(-1, keepdim=True).log() - x.amax(-1, keepdim=True)
    only = torch.full_like(x[:1], -math.inf)
    only[:, s["eos"]] = 0  # a finished beam continues with itself alone
    x = torch.where(s["finished"].bool()[:, None], only, x)
    x = (x + s["scores"].double()[:, None]).reshape(g, w * v)
    best, at = torch.sort(x, dim=-1, descending=True, stable=True)
    best, at = best[:, :s["select"]], at[:, :s["select"]]
    parent, token = at // v, at % v
    ended = s["finished"].reshape(g, w).gather(1, parent).bool() | (token == s["eos"])
    return [parent.reshape(-1).int(), token.reshape(-1).int(), best.reshape(-1).float(),
            ended.reshape(-1).int()]


def _sources(s):
    first = torch.arange(s["groups"], device="cuda")[:, None] * s["beams"]
    return (s["parent"].reshape(s["groups"], s["beams"]) + first).reshape(-1).long()


def _plain_rows(s):
    s["rows"].copy_(s["rows"][:, _sources(s)])
    return s["rows"]


def _plain_pages(s):
    ps, src = s["page"], _sources(s)
    rows = torch.arange(src.numel(), device="cuda")
    held = s["len"].repeat_interleave(s["beams"])
    full, rest = (held // ps).long(), held % ps
    col = full.clamp(max=s["table"].shape[1] - 1)
    copied = (src != rows) & (rest > 0)
    page, spare = s["table"].gather(1, col[:, None])[:, 0], s["spare"].clone()
    a, b = page[src].long(), spare.long()
    part = (torch.arange(ps, device="cuda") < (rest + 7)[:, None] // 8 * 8) & copied[:, None]
    k, v = s["k"], s["v"]
    k[:, b] = torch.where(part[None, :, None, None, :, None], k[:, a], k[:, b])
    v[:, b] = torch.where(part[:, ::8][None, :, None, :, None, None], v[:, a], v[:, b])
    done = torch.arange(s["table"].shape[1], device="cuda") < full[:, None]
    table = torch.where(done, s["table"][src], s["table"])
    own_page = torch.where(copied, spare, table.gather(1, col[:, None])[:, 0])
    s["table"].copy_(table.scatter(1, col[:, None], own_page[:, None]))
    s["spare"].copy_(torch.where(copied, page, spare))
    return [s["table"], s["spare"], k, v]


# ---------------------------------------------------------------- run, own
def _call(s):
    """The framework's function for a state and its arguments: what a program
    sets up once beside its buffers."""
    from synapse_amd import hip
    hip.init(0)
    lib, at = hip.lib(), lambda n: None if s[n] is None else s[n].data_ptr()
    ref = lambda x: (x, ctypes.byref(x))[1]
    if "heads" in s:
        nh, kv, hd = HEADS[s["heads"]]
        pages = ref(hip.KvPages(KV_CODE[s["dtype"]], s["page"], s["k"].shape[1], s["k"].shape[0], kv,
                                hd, at("k"), at("v")))
    if s["kind"] == "append":
        ld = (nh + 2 * kv) * hd
        p = ref(hip.KvAppend(layer=0, n_heads=nh, n_seqs=s["seqs"], rotary_dim=hd, interleaved=0,
                             n_positions=s["cos"].shape[0], eps=1e-6, ldq=ld, ldk=ld, ldv=ld,
                             ldo=nh * hd, ld_table=s["table"].shape[1]))
        q = at("qkv")
        args = (pages, p, s["tokens"], q, q + 4 * nh * hd, q + 4 * (nh + kv) * hd, at("qn"), at("kn"),
                at("cos"), at("sin"), at("pos"), at("seq"), at("index"), at("table"), at("out"), None)
        return lib.syn_hip_kv_append, args, [s["out"], s["k"], s["v"]]
    if s["kind"] == "attend":
        p = ref(hip.PrefixAttention(layer=0, n_heads=nh, n_groups=s["groups"],
                                    group_size=s["members"], max_prefix=s["prefix"],
                                    max_suffix=s["suffix"], scale=0.0, ldq=nh * hd, ldo=nh * hd,
                                    ld_prefix_table=s["ptable"].shape[1],
                                    ld_table=s["table"].shape[1]))
        args = (pages, p, at("q"), at("ptable"), at("plen"), at("table"), at("slen"), at("out"),
                at("scratch"), s["scratch"].numel(), None)
        return lib.syn_hip_prefix_attention, args, s["out"]
    if s["kind"] == "select":
        p = ref(hip.BeamSelect(n_groups=s["groups"], n_beams=s["beams"], n_select=s["select"],
                               eos=s["eos"], pad=s["eos"], vocab=s["vocab"], ld_logits=s["vocab"]))
        args = (p, at("logits"), at("scores"), at("finished"), at("parent"), at("token"), at("score"),
                at("ended"), at("scratch"), s["scratch"].numel(), None)
        return lib.syn_hip_beam_select, args, [s["parent"], s["token"], s["score"], s["ended"]]
    if s["kind"] == "rows":
        n = s["groups"] * s["beams"]
        args = (s["groups"], s["beams"], at("parent"), at("rows"), s["row"], s["row"], s["buffers"],
                n * s["row"], None)
        return lib.syn_hip_beam_reorder_rows, args, s["rows"]
    args = (pages, s["groups"], s["beams"], at("parent"), at("len"), at("table"),
            s["table"].shape[1], at("spare"), None)
    return lib.syn_hip_beam_reorder_pages, args, [s["table"], s["spare"], s["k"], s["v"]]


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        function, args, out = state["call"]
        if function(*args):
            raise RuntimeError("refused: " + state["kind"])
        return out
    return {"append": _plain_append, "attend": _plain_attend, "select": _plain_select,
            "rows": _plain_rows, "pages": _plain_pages}[state["kind"]](state)


# ---------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "select":
        live = c["groups"] * (c["beams"] - c["done"])
        return {"bytes": 4 * live * c["vocab"] + 16 * c["groups"] * c["select"],
                "flops": 4 * live * c["vocab"]}
    if c["kind"] == "rows":  # half of the rows are replaced, from at most as many
        moved = c["beams"] // 2
        return {"bytes": 2 * c["buffers"] * c["groups"] * moved * c["row"], "flops": 0}
    nh, kv, hd = HEADS[c["heads"]]
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "append":
        t = c["tokens"]
        return {"bytes": t * (nh + 2 * kv) * hd * 4 + t * nh * hd * 4 + 2 * (t - c["pad"]) * kv * hd * size,
                "flops": 3 * t * (nh + kv) * hd}
    if c["kind"] == "attend":  # shorter prefixes and suffixes have three quarters of the length on average
        rows = c["groups"] * c["members"]
        prefix = c["prefix"] * (1 + 0.75 * (c["groups"] - 1))
        suffix = c["suffix"] * (1 + 0.75 * (rows - 1))
        return {"bytes": 2 * (prefix + suffix) * kv * hd * size + 8 * rows * nh * hd,
                "flops": 4 * nh * hd * (prefix * c["members"] + suffix)}
    moved = c["groups"] * (c["beams"] // 2)
    part = -(-(c["held"] % c["page"]) // 8) * 8
    return {"bytes": 2 * moved * c["layers"] * 2 * part * kv * hd * size
            + 8 * c["groups"] * c["beams"] * c["room"] // c["page"], "flops": 0}


# ---------------------------------------------------------------- exact
def _flat(pool, page, head, position, dim, tall):
    """elements of layer 0 by page, head, position in the page and dim"""
    _, _, kv, x, y, _ = pool.shape
    hd, ps = (x * 8, y) if tall else (y, x * 8)
    in_head = (dim // 8 * ps + position) * 8 + dim % 8 if tall else (position // 8 * hd + dim) * 8 + position % 8
    return (page * kv + head) * (hd * ps) + in_head


def _exact_append(s):
    nh, kv, hd = HEADS[s["heads"]]
    t, n = s["tokens"], s["tokens"] - s["pad"]
    x = s["qkv"].double().reshape(t, nh + 2 * kv, hd)
    heads = x[:, :nh + kv].clone()
    if s["norm"]:
        heads = heads / ((heads ** 2).sum(-1, keepdim=True) / hd + 1e-6).sqrt()
        heads[:, :nh] *= s["qn"].double()
        heads[:, nh:] *= s["kn"].double()
    pairs = torch.stack([heads[..., :hd // 2], heads[..., hd // 2:]], -1).contiguous()
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
    z = torch.view_as_complex(pairs) * turn
    heads = torch.cat([z.real, z.imag], -1)
    index, seq = s["index"][:n].long(), s["seq"][:n].long()
    page = s["table"].reshape(-1)[seq * s["table"].shape[1] + index // s["page"]].long()
    h, d = torch.arange(kv, device="cuda"), torch.arange(hd, device="cuda")
    k, v = s["k"].double(), s["v"].double()
    for pool, new, tall in ((k, heads[:n, nh:], True), (v, x[:n, nh + kv:], False)):
        where = _flat(pool, page[:, None, None], h[:, None], (index % s["page"])[:, None, None], d, tall)
        pool.reshape(-1)[where.reshape(-1)] = new.reshape(-1)
    return [heads[:, :nh].reshape(t, nh * hd), k, v]


def _exact_attend(s):
    nh, kv, hd = HEADS[s["heads"]]
    out = torch.empty((s["groups"] * s["members"], nh, hd), device="cuda", dtype=torch.float64)
    q = s["q"].double().reshape(-1, nh, hd)
    d = torch.arange(hd, device="cuda")

    def fetch(pages, length, head):
        j = torch.arange(length, device="cuda")[:, None]
        page = pages.long()[j // s["page"]]
        return (s["k"].reshape(-1)[_flat(s["k"], page, head, j % s["page"], d, True)].double(),
                s["v"].reshape(-1)[_flat(s["v"], page, head, j % s["page"], d, False)].double())

    plen, slen = s["plen"].tolist(), s["slen"].tolist()
    for g in range(s["groups"]):
        for h in range(kv):
            heads = slice(h * (nh // kv), (h + 1) * (nh // kv))
            pk, pv = fetch(s["ptable"][g], plen[g], h)
            r = slice(g * s["members"], (g + 1) * s["members"])
            pre = torch.einsum("mad,jd->maj", q[r, heads], pk) / math.sqrt(hd)
            for i in range(s["members"]):
                row = g * s["members"] + i
                sk, sv = fetch(s["table"][row], slen[row], h)
                e = torch.cat([pre[i], q[row, heads] @ sk.T / math.sqrt(hd)], 1)
                p = torch.softmax(e, 1)
                out[row, heads] = p[:, :plen[g]] @ pv + p[:, plen[g]:] @ sv
    return out.reshape(-1, nh * hd)


def _exact_select(s):
    w, best = s["beams"], []
    scores, finished = s["scores"].double().tolist(), s["finished"].tolist()
    for g in range(s["groups"]):
        found = []
        for b in range(g * w, (g + 1) * w):
            if finished[b]:
                found.append(scores[b])
                continue
            logp = torch.log_softmax(s["logits"][b].double(), 0)
            found += (logp.topk(min(s["select"], s["vocab"]))[0] + scores[b]).tolist()
        best += sorted(found, reverse=True)[:s["select"]]
    return [None, None, torch.tensor(best, dtype=torch.float64), None]


def _exact_rows(s):
    rows, parent = s["rows"].double(), s["parent"].tolist()
    out = [rows[:, b // s["beams"] * s["beams"] + p] for b, p in enumerate(parent)]
    return torch.stack(out, 1)


def _exact_pages(s):
    k, v = s["k"].double(), s["v"].double()
    table, spare = s["table"].tolist(), s["spare"].tolist()
    held, parent = s["len"].tolist(), s["parent"].tolist()
    for b, p in enumerate(parent):
        n = held[b // s["beams"]]
        p += b // s["beams"] * s["beams"]
        if p != b and n % s["page"]:
            part, src = -(-(n % s["page"]) // 8), table[p][n // s["page"]]
            k[:, spare[b], :, :, :8 * part] = s["k"][:, src, :, :, :8 * part].double()
            v[:, spare[b], :, :part] = s["v"][:, src, :, :part].double()
    return [None, None, k, v]


def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend, "select": _exact_select,
            "rows": _exact_rows, "pages": _exact_pages}[case["kind"]](prepare(case, seed))
