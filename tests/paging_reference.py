"""Beams, pages and windowed attention in 64 bits, written from their definitions, for the tests."""
from __future__ import annotations

import numpy as np

import low_bit_reference as ref

PAGE, BLOCK = ref.PAGE, ref.BLOCK
BAD_ROWS, NOT_FINITE, NO_PAGES = 1, 2, 4


# ------------------------------------------------------------ attention ----


def window_attention(cache, query, offsets, context, q_heads, sinks, window, out):
    """Rows in 64 bits (others as `out` has them) and the bound of low_bit_reference.attention over the keys that a row
    attends: its sum has at most as many terms as that one counts."""
    d, group = cache.d, q_heads // cache.kv_heads
    o, bound = out.astype(np.float64).copy(), np.zeros(out.shape)
    for s in range(cache.seqs):
        n = offsets[s + 1] - offsets[s]
        if n == 0:
            continue
        for h in range(cache.kv_heads):
            k, v = cache.rows(s, context[s] + n, h)
            for i in range(n):
                p, r = context[s] + i, offsets[s] + i
                j = np.arange(p + 1)
                j = j[(j < sinks) | (p - j < window)]
                for head in range(h * group, (h + 1) * group):
                    at = slice(head * d, (head + 1) * d)
                    q = query[r, at].astype(np.float64)
                    score = k[j] @ q / np.sqrt(d)
                    size = (np.abs(k[j]) @ np.abs(q) / np.sqrt(d)).max() * 1.4427
                    w = np.exp(score - score.max())
                    o[r, at] = w @ v[j] / w.sum()
                    steps = 8 * size + 2 + 16 * (len(j) // PAGE + 3) + 32
                    bound[r, at] = 2 * steps * 2.0 ** -24 * np.abs(v[j]).max()
    return o, bound


# ---------------------------------------------------------------- pages ----


class Pool:
    """Host copy of the pages of several layers, of any content, under one table."""

    NAMES = ("keys", "values", "key_exps", "value_exps")

    def __init__(self, rng, layers, pages, seqs, per_seq, kv_heads, d):
        def random(*shape):
            return rng.integers(-128, 128, (layers, pages, kv_heads, *shape)).astype(np.int8)

        self.keys, self.values = random(PAGE, d), random(d, PAGE)
        self.key_exps, self.value_exps = random(PAGE // BLOCK), random(PAGE // BLOCK)
        self.table, self.users = np.full((seqs, per_seq), -1, np.int32), np.zeros(pages, np.int32)
        self.layers, self.pages, self.seqs, self.per_seq, self.kv_heads, self.d = (layers, pages, seqs, per_seq,
                                                                                  kv_heads, d)

    def fill(self, rng, tokens, share=0.0):
        """Gives sequence s pages for its tokens, in any order; of them a part from the sequence before."""
        order = list(rng.permutation(self.pages))
        for s, n in enumerate(tokens):
            for p in range(-(-n // PAGE)):
                same = s > 0 and self.table[s - 1, p] >= 0 and rng.random() < share
                self.table[s, p] = self.table[s - 1, p] if same else order.pop()
                self.users[self.table[s, p]] += 1

    def upload(self, mmr):
        """Kv8Layers, the table and the users on the device."""
        table, users = mmr.DeviceArray.from_numpy(self.table), mmr.DeviceArray.from_numpy(self.users)
        self.device = [[mmr.DeviceArray.from_numpy(getattr(self, n)[layer]) for n in self.NAMES]
                       for layer in range(self.layers)]
        layers = mmr.Kv8Layers(mmr.Kv8Pages(*parts, table, self.pages, self.seqs, self.per_seq, self.kv_heads, self.d)
                               for parts in self.device)
        return layers, table, users

    def assert_pages_equal(self):
        for layer, parts in enumerate(self.device):
            for name, part in zip(self.NAMES, parts):
                np.testing.assert_array_equal(part.numpy(), getattr(self, name)[layer], err_msg=f"{name} of {layer}")

    def copy(self, source, target, blocks=PAGE // BLOCK):
        n = blocks * BLOCK
        self.keys[:, target, :, :n] = self.keys[:, source, :, :n]
        self.values[:, target, :, :, :n] = self.values[:, source, :, :, :n]
        for e in (self.key_exps, self.value_exps):
            e[:, target, :, :blocks] = e[:, source, :, :blocks]


def fork(pool, parent, keep, room, sinks=0, window=0):
    """In place; returns the error bits."""
    error, before, users = 0, pool.table.copy(), pool.users
    table = np.full_like(before, -1)
    plans = []
    for s in range(pool.seqs):
        p, k, r = int(parent[s]), int(keep[s]), int(room[s])
        if not -1 <= p < pool.seqs or k < 0 or r < 0 or k + r > pool.per_seq * PAGE:
            p, k, r, error = -1, 0, 0, error | BAD_ROWS
        plans.append((p, k if p >= 0 else 0, r))
    for row in before:
        for p in row:
            if 0 <= p < pool.pages:
                users[p] -= 1
    writers = {}
    for s, (p, k, r) in enumerate(plans):
        for place in range(-(-k // PAGE)):
            page = before[p, place]
            behind = window > 0 and place * PAGE >= sinks and place * PAGE + PAGE - 1 < k - window + 1
            if not behind and 0 <= page < pool.pages:
                table[s, place] = page
                users[page] += 1
        if k % PAGE:
            page = table[s, k // PAGE]
            if page < 0:
                error |= BAD_ROWS
            elif r > 0:
                writers.setdefault(page, []).append(s)
    copies = {}
    for page, who in writers.items():
        alone = users[page] == len(who)
        for s in who[1:] if alone else who:
            copies[s] = page
            users[page] -= 1
            table[s, plans[s][1] // PAGE] = -1
    free = [p for p in range(pool.pages) if users[p] <= 0]
    for s, (p, k, r) in enumerate(plans):
        for place in range(k // PAGE, -(-(k + r) // PAGE)):
            if table[s, place] >= 0:
                continue
            if not free:
                error |= NO_PAGES
                continue
            page = table[s, place] = free.pop(0)
            users[page] = 1
            if s in copies and place == k // PAGE:
                pool.copy(copies[s], page, -(-(k % PAGE) // BLOCK))
    pool.table = table
    return error


def compact(pool):
    """In place; returns each page's new number and how many are in use."""
    used = pool.users > 0
    live = int(used.sum())
    holes = [p for p in range(live) if not used[p]]
    moved = np.where(used, np.arange(pool.pages), -1).astype(np.int32)
    for source, hole in zip([p for p in range(live, pool.pages) if used[p]], holes):
        moved[source] = hole
        pool.copy(source, hole)
        pool.users[hole], pool.users[source] = pool.users[source], 0
    held = (pool.table >= 0) & (pool.table < pool.pages)
    pool.table = np.where(held, moved[np.where(held, pool.table, 0)], -1).astype(np.int32)
    return moved, live


# ---------------------------------------------------------------- beams ----


def select(logits, beams, eos, power, scores, lengths, ended):
    """The candidates chosen: (scores in 64 bits, lengths, ended, parent, token), the error bits, and what scores may be
    off by without another choice: of one that was chosen and the next (of another beam and not of equal rank), the gap
    of their ranks over what an error of 1 of both scores makes of it."""
    rows, vocab = logits.shape
    out = [np.full(rows, -np.inf), np.zeros(rows, np.int32), np.full(rows, int(eos >= 0), np.int32),
           np.full(rows, -1, np.int32), np.full(rows, max(eos, 0), np.int32)]
    error, gap = 0, np.inf
    for first in range(0, rows, beams):
        rank, score, row, token, x, factor = [], [], [], [], [], {}
        for b in range(first, first + beams):
            done = eos >= 0 and ended[b] != 0
            length = max(int(lengths[b]) + (0 if done else 1), 1)
            values = logits[b].astype(np.float64)
            bad = not scores[b] < np.inf or (not done and not (values < np.inf).all())
            error |= NOT_FINITE if bad else 0
            if bad or scores[b] == -np.inf:
                continue
            if done:
                s, t, values = np.array([float(scores[b])]), np.array([eos]), np.zeros(1)
            else:
                top = values.max()
                if top == -np.inf:
                    continue
                s = float(scores[b]) + (values - (top + np.log(np.exp(values - top).sum())))
                t = np.arange(vocab)
            with np.errstate(over="ignore"):
                fine = s.astype(np.float32) > -np.inf
            factor[b] = float(length) ** -power
            rank.append(s[fine] * factor[b])
            score.append(s[fine]), token.append(t[fine]), x.append(values[fine])
            row.append(np.full(fine.sum(), b))
        if not rank:
            continue
        rank, score, row, token, x = (np.concatenate(a) for a in (rank, score, row, token, x))
        order = np.lexsort((token, -x, row, -rank))[: beams + 1]
        for a, b in zip(order[:-1], order[1:]):
            if row[a] != row[b] and rank[a] != rank[b]:
                gap = min(gap, (rank[a] - rank[b]) / (factor[row[a]] + factor[row[b]]))
        order = order[:beams]
        to = slice(first, first + len(order))
        out[0][to], out[3][to], out[4][to] = score[order], row[order], token[order]
        done = (ended[row[order]] != 0) & (eos >= 0)
        out[1][to] = lengths[row[order]] + np.where(done, 0, 1)
        out[2][to] = (token[order] == eos) if eos >= 0 else 0
    return out, error, gap
