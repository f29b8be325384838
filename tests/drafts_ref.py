"""Verification of drafts and page tables in plain numpy, for the tests."""
from collections import deque

import numpy as np


# ---------------------------------------------------------------- verification
def softmax(row, heat):
    """float64 probabilities of a row of logits (NaN counts as -inf), zeros where none is above -inf"""
    x = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return np.zeros(len(x))
    if top == np.inf:
        e = (x == np.inf).astype(np.float64)
    else:
        e = np.exp((x - top) / float(heat))
    return e / e.sum()


def verify(target, draft, drafted, n, heat, u, pad, width):
    """one sequence: (tokens [width + 1], count, log-probabilities, how far u was from the
    nearest border of a decision, relative)"""
    tokens, logp = np.full(width + 1, pad, np.int64), np.zeros(width + 1)
    if n < 0:
        return tokens, 0, logp, np.inf
    n = min(n, width)
    near, vocab = np.inf, target.shape[1]
    greedy = not (heat > 0 and np.isfinite(heat))
    for i in range(n + 1):
        row = target[i]
        if greedy:
            x = np.where(np.isnan(row), -np.inf, row)
            best = int(x.argmax()) if x.max() > -np.inf else -1
            if i < n and best >= 0 and drafted[i] == best:
                tokens[i] = best
                continue
            if best >= 0:
                tokens[i] = best
            else:
                logp[i] = -np.inf
            return tokens, i + 1, logp, near
        p = softmax(row, heat)
        weight = p
        if i < n:
            x = int(drafted[i])
            q = np.zeros(vocab)
            if draft is None:
                if x < vocab:
                    q[x] = 1.0
            else:
                q = softmax(draft[i], heat)
            if x < vocab:
                a, b = float(u[i]) * q[x], p[x]
                if max(a, b) > 0:
                    near = min(near, abs(a - b) / max(a, b))
                if a < b:
                    tokens[i], logp[i] = x, np.log(p[x])
                    continue
            weight = np.maximum(p - q, 0.0)
            if not weight.sum() > 0:
                weight = p
        total = weight.sum()
        if not total > 0:
            logp[i] = -np.inf
            return tokens, i + 1, logp, near
        sums = np.cumsum(weight)
        border = float(u[width]) * sums[-1]
        t = int(np.searchsorted(sums, border, side="right"))
        if t >= vocab:
            t = int(np.flatnonzero(weight)[-1])
        near = min(near, abs(sums[t] - border) / sums[-1], (border - (sums[t] - weight[t])) / sums[-1]
                   if weight[t] < sums[t] else np.inf)
        tokens[i], logp[i] = t, np.log(p[t])
        return tokens, i + 1, logp, near
    raise AssertionError


# ---------------------------------------------------------------- page tables
class Tables:
    def __init__(self, page, pages, seqs, cols):
        self.page, self.pages = page, pages
        self.table = np.full((seqs, cols), -1, np.int32)
        self.held = np.zeros(seqs, np.int32)
        self.refs = np.zeros(pages, np.int32)

    def holds(self, s):
        return min(max(int(self.held[s]), 0), self.table.shape[1])

    def give_back(self, s, first):
        for c in range(first, self.holds(s)):
            p = self.table[s, c]
            if 0 <= p < self.pages and self.refs[p] > 0:
                self.refs[p] -= 1
            self.table[s, c] = -1
        self.held[s] = min(self.holds(s), first)

    def take(self, wants):
        """wants: [(row, pages it needs)] in order"""
        free = deque(np.flatnonzero(self.refs == 0).tolist())
        for s, n in wants:
            for _ in range(n):
                if not free:
                    return
                p = free.popleft()
                self.table[s, self.held[s]] = p
                self.held[s] += 1
                self.refs[p] = 1

    def resize(self, lens):
        wants = []
        for s, n in enumerate(lens):
            if n < 0:
                continue
            want = min(-(-int(n) // self.page), self.table.shape[1])
            self.give_back(s, want)
            wants.append((s, max(0, want - int(self.held[s]))))
        self.take(wants)

    def fork(self, parent, lens):
        """returns the copies of parts of pages: [(from, to, positions)]"""
        n = len(parent)
        rows = [s for s in range(n)
                if parent[s] != s and 0 <= parent[s] < n and parent[parent[s]] == parent[s]]
        for s in rows:
            self.give_back(s, 0)
        wants, tails = [], []
        for s in rows:
            p = parent[s]
            length = min(max(int(lens[s]), 0), self.holds(p) * self.page)
            full, rest = length // self.page, length % self.page
            for c in range(full):
                page = self.table[p, c]
                self.table[s, c] = page
                if 0 <= page < self.pages:
                    self.refs[page] += 1
            self.held[s] = full
            wants.append((s, int(rest > 0)))
            if rest:
                tails.append((s, p, full, -(-rest // 8) * 8))
        self.take(wants)
        return [(int(self.table[p, c]), int(self.table[s, c]), m) for s, p, c, m in tails
                if self.held[s] > c and 0 <= self.table[p, c] < self.pages]

    def compact(self, to):
        """into the tables `to`; returns (live pages, [(from, to)])"""
        live = np.flatnonzero(self.refs > 0)
        number = np.full(self.pages, -1, np.int64)
        number[live] = np.arange(len(live))
        number[number >= to.pages] = -1
        to.refs[:] = 0
        kept = live[:to.pages]
        to.refs[:len(kept)] = self.refs[kept]
        to.table[:] = -1
        for s in range(len(self.held)):
            to.held[s] = self.holds(s)
            for c in range(self.holds(s)):
                p = self.table[s, c]
                if 0 <= p < self.pages:
                    to.table[s, c] = number[p]
        return len(live), list(zip(kept.tolist(), range(len(kept))))
