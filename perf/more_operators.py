"""Sampling with drafted tokens over a paged cache: the operators, as cases to be timed.

- ``attend``: causal attention of several new tokens of each sequence over its
  pages: one token (decoding), a few (drafts to be verified), many (a prompt's
  chunk) (``syn_hip_paged_attention``).
- ``verify``: drafted tokens against the target's probabilities, from given
  random numbers, and the token after them (``syn_hip_draft_verify``).
- ``resize``, ``fork``, ``compact``: pages taken and given back, sequences that
  continue another one, live pages moved to another pool (``syn_hip_kv_resize``,
  ``syn_hip_kv_fork``, ``syn_hip_kv_compact``).

A page holds ``page`` positions of one layer's keys as [kv head][dim / 8][position][8]
and values as [kv head][position / 8][dim][8].  A row of a page table holds the
pages of a sequence, ``held`` of them; ``refs`` counts the entries that name a page.
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
        # four samples of a short prompt, four drafts each to verify: latency
        dict(name="attend_drafts_short", kind="attend", heads="qwen", dtype="f32", seqs=4, new=5,
             length=213, window=0, page=16),
        # conversations, one token each: a decode step of a server
        dict(name="attend_tokens", kind="attend", heads="llama1b", dtype="bf16", seqs=64, new=1,
             length=12000, window=0, page=64),
        # conversations with up to seven drafts each
        dict(name="attend_drafts", kind="attend", heads="mistral", dtype="f16", seqs=24, new=8,
             length=8200, window=0, page=16),
        # chunks of two long prompts
        dict(name="attend_chunks", kind="attend", heads="llama3b", dtype="f16", seqs=2, new=1536,
             length=12001, window=0, page=64),
        # one sequence, four drafts, a small vocabulary: latency
        dict(name="verify_one", kind="verify", seqs=1, drafts=4, vocab=32000),
        # a server's batch with eight drafts each
        dict(name="verify_batch", kind="verify", seqs=64, drafts=8, vocab=151936),
        # one step of 16 samples: positions of rejected drafts back, the next ones' taken
        dict(name="resize_step", kind="resize", seqs=16, length=700, by=9, pages=2048, page=16),
        # a large server between two steps, some requests at their end
        dict(name="resize_server", kind="resize", seqs=1024, length=3001, by=1500, pages=262144,
             page=16),
        # eight samples of one prompt, LLaMA-3.2-3B
        dict(name="fork_samples", kind="fork", heads="llama3b", dtype="f32", layers=28, groups=1,
             members=8, length=333, page=16),
        # four samples of each of 32 prompts, Qwen3-0.6B
        dict(name="fork_server", kind="fork", heads="qwen", dtype="bf16", layers=28, groups=32,
             members=4, length=1500, page=64),
        # what eight short requests hold, to a smaller pool
        dict(name="compact_small", kind="compact", heads="lfm", dtype="f32", layers=6, seqs=8,
             length=150, pages=200, page=16),
        # a server's cache to a larger pool, LLaMA-3.2-3B
        dict(name="compact_server", kind="compact", heads="llama3b", dtype="f16", layers=28, seqs=32,
             length=900, pages=800, page=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("attend", "verify", "resize", "fork", "compact"), (8, 6, 3, 3, 2))[0]
    heads, dtype = rng.choice(sorted(HEADS)), rng.choice(sorted(DTYPE))
    page = rng.choice((8, 16, 32, 64, 128))
    if kind == "attend":
        new = rng.choice((1, rng.randrange(2, 10), _log_int(rng, 10, 1536)))
        c = dict(kind=kind, heads=heads, dtype=dtype, seqs=_log_int(rng, 1, 64), new=new,
                 length=new + _log_int(rng, 1, 32768),
                 window=rng.choice((0, 0, 0, _log_int(rng, 16, 4096))), page=page)
        while (work(c)["bytes"] > 1e9 or work(c)["flops"] > 3e11
               or c["seqs"] * c["new"] * HEADS[heads][0] * c["length"] > 8e8):
            c["seqs"], c["length"] = max(1, c["seqs"] * 3 // 4), max(new, c["length"] * 3 // 4)
        return c
    if kind == "verify":
        drafts = rng.choice((0, rng.randrange(1, 6), rng.randrange(1, 13)))
        vocab = rng.choice(VOCABS) - (rng.randrange(1, 64) if rng.random() < 0.5 else 0)
        return dict(kind=kind, seqs=_log_int(rng, 1, max(1, 540 // (drafts + 1))), drafts=drafts,
                    vocab=vocab)
    if kind == "resize":
        seqs, length = _log_int(rng, 1, 1024), _log_int(rng, 20, 4000)
        by = rng.randrange(1, length)
        return dict(kind=kind, seqs=seqs, length=length, by=by, page=page,
                    pages=rng.randrange(1, 3) * seqs * _up(length, page) + rng.randrange(1, 99))
    layers = rng.randrange(1, 17)
    if kind == "fork":
        return dict(kind=kind, heads=heads, dtype=dtype, layers=layers,
                    groups=rng.randrange(1, 9), members=rng.randrange(2, 9),
                    length=_log_int(rng, 2, 1000), page=page)
    seqs, length = rng.randrange(1, 17), _log_int(rng, 8, 500)
    return dict(kind=kind, heads=heads, dtype=dtype, layers=layers, seqs=seqs, length=length,
                pages=seqs * _up(length, page) + rng.randrange(1, 60), page=page)


def _up(a, b):
    return -(-a // b)


def _news(c):
    """new tokens of each sequence: from the case's down to half of it"""
    return [c["new"] - 5 * i % (c["new"] // 2 + 1) for i in range(c["seqs"])]


# ---------------------------------------------------------------- prepare
def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000 + salt)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


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


def _prepare_attend(c, seed):
    g = _gen(seed)
    nh, kv, hd = HEADS[c["heads"]]
    n, cols = c["seqs"], _up(c["length"], c["page"])
    news = torch.tensor(_news(c), device="cuda", dtype=torch.int32)
    start = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int32), news.cumsum(0).int()])
    k, v = _pool(g, c, 1, n * cols)
    # the longest is the case's; others are up to half shorter
    length = c["length"] - _ints(g, 0, c["length"] // 2 + 1, n)
    length[n // 2] = c["length"]
    tokens = sum(_news(c))
    return dict(c, tokens=tokens, k=k, v=v, q=_randn(g, tokens, nh * hd), start=start,
                len=torch.maximum(length, news), table=_pages(g, n * cols, n, cols),
                out=torch.zeros((tokens, nh * hd), device="cuda"),
                # scratch of the split attention: as much as any split of this work may ask for
                scratch=torch.empty(256 << 20, device="cuda", dtype=torch.uint8))


def _prepare_verify(c, seed):
    g = _gen(seed)
    n, d, vocab = c["seqs"], c["drafts"], c["vocab"]
    draft = _randn(g, n, max(d, 1), vocab) * 2.5
    target = _randn(g, n, d + 1, vocab)
    # a draft model that is right more often than not
    target[:, :d] = draft[:, :d] + 0.5 * target[:, :d]
    target[:, d] *= 2.5
    target[..., ::1009], draft[..., ::1009] = -math.inf, -math.inf  # words that the caller bans
    heat = 0.6 + 0.6 * torch.rand(n, generator=g, device="cuda")
    heat[3::8] = 0  # greedy requests
    some = -torch.log(-torch.log(torch.rand((n, max(d, 1), vocab), generator=g, device="cuda")))
    token = (draft + heat[:, None, None] * some).argmax(-1).int()  # drawn from the draft's softmax
    count = d - _ints(g, 0, d // 2 + 1, n)
    count[0] = d
    return dict(c, target=target, draft=draft, token=token, count=count, heat=heat,
                u=torch.rand((n, d + 1), generator=g, device="cuda"),
                out=torch.zeros((n, d + 1), device="cuda", dtype=torch.int32),
                emitted=torch.zeros(n, device="cuda", dtype=torch.int32),
                logp=torch.zeros((n, d + 1), device="cuda"),
                scratch=torch.empty(16 << 20, device="cuda", dtype=torch.uint8))


def _tables(g, pages, held, cols):
    """rows of distinct pages, in no order, -1 behind the held ones; and the counts"""
    ids = _pages(g, pages, held.numel(), cols)
    on = torch.arange(cols, device="cuda") < held[:, None]
    table = torch.where(on, ids, -1)
    refs = torch.zeros(pages, device="cuda", dtype=torch.int32)
    refs[ids[on].long()] = 1
    return dict(table=table, held=held.clone(), refs=refs,
                scratch=torch.empty(16 << 20, device="cuda", dtype=torch.uint8))


def _prepare_resize(c, seed):
    g = _gen(seed)
    n, page = c["seqs"], c["page"]
    long = c["length"] - _ints(g, 0, c["length"] // 2 + 1, n)
    short = (long - _ints(g, 0, c["by"] + 1, n)).clamp(min=0)
    held = ((long + page - 1) // page).int()
    return dict(c, short=short, long=long, **_tables(g, c["pages"], held, _up(c["length"], page)))


def _prepare_fork(c, seed):
    g = _gen(seed)
    rows, cols, page = c["groups"] * c["members"], _up(c["length"], c["page"]), c["page"]
    length = c["length"] - _ints(g, 0, c["length"] // 2 + 1, c["groups"])
    length[0] = c["length"]
    length = length.repeat_interleave(c["members"])
    row = torch.arange(rows, device="cuda", dtype=torch.int32)
    first = row // c["members"] * c["members"]
    # what the last samples of these rows held goes back
    held = torch.where(row == first, (length + page - 1) // page, _ints(g, 0, cols + 1, rows)).int()
    k, v = _pool(g, c, c["layers"], rows * cols)
    return dict(c, k=k, v=v, parent=first, len=length, **_tables(g, rows * cols, held, cols))


def _prepare_compact(c, seed):
    g = _gen(seed)
    n, cols, page = c["seqs"], _up(c["length"], c["page"]), c["page"]
    held = torch.full((n,), cols, device="cuda", dtype=torch.int32)
    k, v = _pool(g, c, c["layers"], c["pages"])
    to_pages = n * cols + 7
    zeros = lambda *shape: torch.zeros(shape, device="cuda", dtype=torch.int32)
    return dict(c, k=k, v=v, **_tables(g, c["pages"], held, cols),
                to_pages=to_pages, to_k=torch.zeros_like(k[:, :1]).repeat(1, to_pages, 1, 1, 1, 1),
                to_v=torch.zeros_like(v[:, :1]).repeat(1, to_pages, 1, 1, 1, 1), to_table=zeros(n, cols),
                to_held=zeros(n), to_refs=zeros(to_pages), live=zeros(1))


def prepare(case, seed):
    return {"attend": _prepare_attend, "verify": _prepare_verify, "resize": _prepare_resize,
            "fork": _prepare_fork, "compact": _prepare_compact}[case["kind"]](dict(case), seed)


# ---------------------------------------------------------------- run, plain
def _keys(s, table):
    """[table rows, kv head, position, dim] in float32"""
    x = s["k"][0][table.long()].float()  # rows, pages, kv, dim / 8, position, 8
    return x.permute(0, 2, 1, 4, 3, 5).flatten(4, 5).flatten(2, 3)


def _values(s, table):
    x = s["v"][0][table.long()].float()  # rows, pages, kv, position / 8, dim, 8
    return x.permute(0, 2, 1, 3, 5, 4).flatten(2, 4)


def _plain_attend(s):
    nh, kv, hd = HEADS[s["heads"]]
    n, new, rep = s["seqs"], s["new"], nh // kv
    start, count = s["start"][:-1].long(), (s["start"][1:] - s["start"][:-1]).long()
    j = torch.arange(new, device="cuda")
    row = (start[:, None] + j).clamp(max=s["tokens"] - 1)
    q = s["q"][row].reshape(n, new, kv, rep, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, new * rep, hd)
    x = q @ _keys(s, s["table"]).transpose(-1, -2).contiguous() * (1 / math.sqrt(hd))
    last = s["len"].long()[:, None] - count[:, None] + j  # the last position that a token sees
    at = torch.arange(x.shape[-1], device="cuda")
    off = at > last[..., None]
    if s["window"]:
        off |= at <= last[..., None] - s["window"]
    x = x.reshape(n, kv, new, rep, -1).masked_fill_(off[:, None, :, None], -math.inf)
    x = torch.exp_(x.sub_(x.amax(-1, keepdim=True).clamp(min=-1e30)))
    total = x.sum(-1, keepdim=True)
    out = (x.reshape(n, kv, new * rep, -1) @ _values(s, s["table"])).reshape(n, kv, new, rep, hd)
    out = torch.where(total > 0, out / total, 0).permute(0, 2, 1, 3, 4).reshape(n, new, nh * hd)
    s["out"][row[j < count[:, None]]] = out[j < count[:, None]]
    return s["out"]


def _plain_verify(s):
    n, d, vocab = s["seqs"], s["drafts"], s["vocab"]
    i, rows = torch.arange(d + 1, device="cuda"), torch.arange(n, device="cuda")
    greedy = (s["heat"] <= 0)[:, None, None]
    heat = torch.where(greedy, 1, s["heat"][:, None, None]).double()

    def logs(x):  # in 64 bits: a draw may fall next to a border between two tokens
        x = x.double() / heat
        x = x - x.amax(-1, keepdim=True)
        x = x - x.exp().sum(-1, keepdim=True).log()
        return x

    lp = logs(s["target"])
    lq = logs(s["draft"]) if d else lp
    best = s["target"].argmax(-1)
    token = s["token"][:, :d].long()
    p = lp[:, :d].gather(-1, token[..., None])[..., 0].exp()
    q = lq[:, :d].gather(-1, token[..., None])[..., 0].exp()
    fine = torch.where(greedy[..., 0], token == best[:, :d], s["u"][:, :d].double() * q < p)
    fine &= i[:d] < s["count"][:, None]
    r = fine.int().cumprod(-1).sum(-1)  # drafts accepted
    p = lp[rows, r].exp()
    rest = (p - lq[rows, r.clamp(max=max(d - 1, 0))].exp()).clamp(min=0)
    rest = torch.where((r < s["count"])[:, None], rest, p)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
    upto = rest.cumsum(-1)
    chosen = (upto <= s["u"][:, d:].double() * upto[:, -1:]).sum(-1)
    final = vocab - 1 - (rest > 0).flip(-1).int().argmax(-1)
    chosen = torch.where(greedy[:, 0, 0], best[rows, r], torch.minimum(chosen, final))
    out = torch.cat([s["token"][:, :d].long(), torch.zeros_like(chosen)[:, None]], 1)
    out = torch.where(i < r[:, None], out, 0).scatter(1, r[:, None], chosen[:, None])
    logp = lp.gather(-1, out[..., None])[..., 0]
    logp = torch.where((i <= r[:, None]) & ~greedy[..., 0], logp, 0)
    return [out.int(), (r + 1).int(), logp.float()]


def _take(s, keep, want):
    """Rows keep their first ``keep`` entries; the free pages of lowest number go
    to the entries from there to ``want``, in order"""
    table, held, refs = s["table"], s["held"], s["refs"]
    col = torch.arange(table.shape[1], device="cuda")
    give = (col >= keep[:, None]) & (col < held[:, None])
    gone = table[give].long()
    refs.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    table.masked_fill_(give, -1)
    free = (refs == 0).nonzero()[:, 0].int()
    need = (col >= keep[:, None]) & (col < want[:, None])
    rank = need.reshape(-1).cumsum(0).reshape(need.shape)
    need &= rank <= free.numel()
    pages = free[:int(need.sum())]
    table.masked_scatter_(need, pages)
    refs[pages.long()] = 1
    held.copy_(keep + need.sum(-1))
    return need


def _plain_resize(s):
    for length in (s["short"], s["long"]):
        want = (length + s["page"] - 1) // s["page"]
        _take(s, torch.minimum(s["held"], want), want)
    return [s["table"], s["held"], s["refs"]]


def _plain_fork(s):
    page, parent = s["page"], s["parent"].long()
    rows = torch.arange(parent.numel(), device="cuda")
    child = parent != rows
    full, rest = s["len"] // page, s["len"] % page
    keep = torch.where(child, 0, s["held"])
    _take(s, keep, keep)  # what the children held
    col = torch.arange(s["table"].shape[1], device="cuda")
    shared = (col < full[:, None]) & child[:, None]
    s["table"].copy_(torch.where(shared, s["table"][parent], s["table"]))
    names = s["table"][shared].long()
    s["refs"].index_add_(0, names, torch.ones_like(names, dtype=torch.int32))
    keep = torch.where(child, full, s["held"])
    s["held"].copy_(keep)
    _take(s, keep, keep + (child & (rest > 0)).int())
    copied = child & (s["held"] > full)
    at = full.clamp(max=s["table"].shape[1] - 1).long()[:, None]
    a = s["table"][parent].gather(1, at)[:, 0][copied].long()
    b = s["table"].gather(1, at)[:, 0][copied].long()
    part = torch.arange(page, device="cuda") < (rest[copied] + 7)[:, None] // 8 * 8
    k, v = s["k"], s["v"]
    k[:, b] = torch.where(part[None, :, None, None, :, None], k[:, a], k[:, b])
    v[:, b] = torch.where(part[:, ::8][None, :, None, :, None, None], v[:, a], v[:, b])
    return [s["table"], s["held"], s["refs"], k, v]


def _plain_compact(s):
    live = s["refs"] > 0
    new = torch.where(live, live.cumsum(0) - 1, -1).int()
    old = live.nonzero()[:, 0]
    s["live"].copy_(live.sum())
    s["to_k"][:, :old.numel()] = s["k"][:, old]
    s["to_v"][:, :old.numel()] = s["v"][:, old]
    s["to_refs"].zero_()
    s["to_refs"][:old.numel()] = s["refs"][old]
    s["to_held"].copy_(s["held"])
    on = torch.arange(s["table"].shape[1], device="cuda") < s["held"][:, None]
    s["to_table"].copy_(torch.where(on, new[s["table"].clamp(min=0).long()], -1))
    return [s["live"], s["to_table"], s["to_held"], s["to_refs"], s["to_k"], s["to_v"]]


# ---------------------------------------------------------------- run, own
def _call(s):
    """The framework's functions for a state and their arguments: what a program
    sets up once beside its buffers."""
    from synapse_amd import hip
    hip.init(0)
    lib, at = hip.lib(), lambda n: s[n].data_ptr()
    ref = lambda x: (x, ctypes.byref(x))[1]
    scratch = (at("scratch"), s["scratch"].numel(), None)

    def pages(pre=""):
        _, kv, hd = HEADS[s["heads"]]
        return ref(hip.KvPages(KV_CODE[s["dtype"]], s["page"], s[pre + "k"].shape[1],
                               s[pre + "k"].shape[0], kv, hd, at(pre + "k"), at(pre + "v")))

    def tables(pre=""):
        t = s[pre + "table"]
        return ref(hip.KvTables(page_size=s["page"], n_pages=s[pre + "refs"].numel(), n_seqs=t.shape[0],
                                ld_table=t.shape[1], table=at(pre + "table"), held=at(pre + "held"),
                                refs=at(pre + "refs")))

    if s["kind"] == "attend":
        nh, _, hd = HEADS[s["heads"]]
        p = ref(hip.PagedAttention(layer=0, n_heads=nh, n_seqs=s["seqs"], n_tokens=s["tokens"],
                                   max_new=s["new"], max_len=s["length"], window=s["window"], scale=0.0,
                                   ldq=nh * hd, ldo=nh * hd, ld_table=s["table"].shape[1]))
        args = (pages(), p, at("q"), at("start"), at("len"), at("table"), at("out")) + scratch
        return [(lib.syn_hip_paged_attention, args)], s["out"]
    if s["kind"] == "verify":
        d, v = s["drafts"], s["vocab"]
        p = ref(hip.DraftVerify(n_seqs=s["seqs"], max_draft=d, pad=0, vocab=v, ld_target=v,
                                target_stride=(d + 1) * v, ld_draft=v, draft_stride=max(d, 1) * v))
        args = (p, at("target"), at("draft"), at("token"), at("count"), at("heat"), at("u"), at("out"),
                at("emitted"), at("logp")) + scratch
        return [(lib.syn_hip_draft_verify, args)], [s["out"], s["emitted"], s["logp"]]
    out = [s["table"], s["held"], s["refs"]]
    if s["kind"] == "resize":
        return [(lib.syn_hip_kv_resize, (tables(), at(n)) + scratch) for n in ("short", "long")], out
    if s["kind"] == "fork":
        args = (pages(), tables(), at("parent"), at("len")) + scratch
        return [(lib.syn_hip_kv_fork, args)], out + [s["k"], s["v"]]
    args = (pages(), tables(), pages("to_"), tables("to_"), at("live")) + scratch
    return [(lib.syn_hip_kv_compact, args)], [s[n] for n in ("live", "to_table", "to_held", "to_refs",
                                                             "to_k", "to_v")]


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        calls, out = state["call"]
        for function, args in calls:
            if function(*args):
                raise RuntimeError("refused: " + state["kind"])
        return out
    return {"attend": _plain_attend, "verify": _plain_verify, "resize": _plain_resize,
            "fork": _plain_fork, "compact": _plain_compact}[state["kind"]](state)


# ---------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "attend":  # shorter sequences have three quarters of the length on average
        nh, kv, hd = HEADS[c["heads"]]
        size, bytes_, flops = (4 if c["dtype"] == "f32" else 2), 0, 0
        for i, n in enumerate(_news(c)):
            length = c["length"] if i == c["seqs"] // 2 else max(n, 0.75 * c["length"])
            seen = min(length, c["window"] + n) if c["window"] else length
            each = min(length - n / 2, c["window"]) if c["window"] else length - n / 2
            bytes_ += 2 * seen * kv * hd * size + 8 * n * nh * hd
            flops += 4 * nh * hd * n * each
        return {"bytes": bytes_, "flops": flops}
    if c["kind"] == "verify":  # a quarter of the drafts is not there on average
        n, d = c["seqs"], 0.75 * c["drafts"]
        return {"bytes": 4 * n * (2 * d + 1) * c["vocab"], "flops": 4 * n * (2 * d + 1) * c["vocab"]}
    if c["kind"] == "resize":  # the counts, and each changed entry and its count twice
        return {"bytes": 8 * c["pages"] + 16 * c["seqs"] * c["by"] / 2 / c["page"] + 32 * c["seqs"],
                "flops": 0}
    _, kv, hd = HEADS[c["heads"]]
    place = 2 * kv * hd * (4 if c["dtype"] == "f32" else 2) * c["layers"]  # one position
    if c["kind"] == "fork":
        rows = c["groups"] * (c["members"] - 1)
        # the first group's length is the case's, the others' last pages are half full on average
        first = _up(c["length"] % c["page"], 8) * 8 * (c["members"] - 1)
        return {"bytes": 2 * place * (first + (rows - c["members"] + 1) * c["page"] / 2)
                + 16 * rows * c["length"] / c["page"], "flops": 0}
    live = c["seqs"] * _up(c["length"], c["page"])
    return {"bytes": 2 * place * live * c["page"] + 8 * live + 8 * c["pages"], "flops": 0}


# ---------------------------------------------------------------- exact
def _exact_attend(s):
    nh, kv, hd = HEADS[s["heads"]]
    rep, page = nh // kv, s["page"]
    out = torch.zeros((s["tokens"], nh, hd), device="cuda", dtype=torch.float64)
    start, length = s["start"].tolist(), s["len"].tolist()
    for i in range(s["seqs"]):
        n, q = start[i + 1] - start[i], s["q"][start[i]:start[i + 1]].double().reshape(-1, nh, hd)
        j = torch.arange(length[i], device="cuda")
        pages = s["table"][i].long()[j // page]
        here = length[i] - n + torch.arange(n, device="cuda")[:, None]
        seen = (j <= here) & ((j > here - s["window"]) if s["window"] else True)
        for h in range(kv):
            k = s["k"][0, pages, h, :, j % page].double().reshape(-1, hd)
            v = s["v"][0, pages, h, j % page // 8, :, j % 8].double()
            for r in range(h * rep, (h + 1) * rep):
                e = (q[:, r] @ k.T / math.sqrt(hd)).masked_fill(~seen, -math.inf)
                out[start[i]:start[i + 1], r] = torch.softmax(e, 1) @ v
    return out.reshape(-1, nh * hd)


def _exact_verify(s):
    logp = torch.zeros((s["seqs"], s["drafts"] + 1), dtype=torch.float64)
    heat, count, token, u = (s[n].tolist() for n in ("heat", "count", "token", "u"))
    for i in range(s["seqs"]):
        if heat[i] <= 0:
            continue  # a token that is certain
        scaled = lambda x: torch.softmax(x.double() / heat[i], -1)
        left = None
        for j in range(count[i] + 1):
            p = scaled(s["target"][i, j])
            if j == count[i]:
                left = p
                break
            q = scaled(s["draft"][i, j])
            x = token[i][j]
            if u[i][j] * q[x].item() >= p[x].item():
                left = torch.relu(p - q)
                break
            logp[i, j] = p[x].log().item()
        x = torch.searchsorted(left.cumsum(0), u[i][-1] * left.sum().item(), right=True).item()
        logp[i, j] = p[min(x, s["vocab"] - 1)].log().item()
    return [None, None, logp]


def _exact_fork(s):
    # the copies depend on the pages taken: those of lowest number that nothing names
    page, cols = s["page"], s["table"].shape[1]
    k, v = s["k"].double(), s["v"].double()
    parent, length, held = (s[n].tolist() for n in ("parent", "len", "held"))
    table, refs = s["table"].tolist(), s["refs"].tolist()
    kids = [r for r in range(len(parent)) if parent[r] != r]
    for r in kids:
        for c in range(held[r]):
            refs[table[r][c]] -= 1
    free = iter([p for p, n in enumerate(refs) if n == 0])
    for r in kids:
        rest = length[r] % page
        if rest and length[r] // page < cols:
            to, src, eight = next(free), table[parent[r]][length[r] // page], _up(rest, 8)
            k[:, to, :, :, :8 * eight] = s["k"][:, src, :, :, :8 * eight].double()
            v[:, to, :, :eight] = s["v"][:, src, :, :eight].double()
    return [None, None, None, k, v]


def _exact_compact(s):
    k, v = s["to_k"].double(), s["to_v"].double()
    for to, src in enumerate(p for p, n in enumerate(s["refs"].tolist()) if n > 0):
        k[:, to], v[:, to] = s["k"][:, src].double(), s["v"][:, src].double()
    return [None, None, None, None, k, v]


def exact(case, seed):
    how = {"attend": _exact_attend, "verify": _exact_verify, "fork": _exact_fork,
           "compact": _exact_compact}.get(case["kind"])
    return how(prepare(case, seed)) if how else None
