"""The 8-bit cache's attention where a wave or a split has so many pages that it reads its page numbers again (64), and
that its int32 sums move to fp32 (1,024): tables that repeat a few pages, against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import low_bit_reference as ref
from test_gpu_kv8 import attend, ints

pytestmark = pytest.mark.gpu
D, KINDS = 32, 5


class Repeated:
    """Sequences whose tables repeat KINDS pages in any order, so that 64 bits need only how often a row meets each.
    One more page is met once, at a place of its own in each table, and the queries aim at a key of it, which takes
    a fair share of a row's weight: a page number read from another place, or a page left out, shows."""

    def __init__(self, mmr, rng, hot_at, per, kv_heads):
        self.cache = c = ref.Cache(rng, KINDS + 1, 1, KINDS + 1, kv_heads, D)
        c.table = np.arange(KINDS + 1, dtype=np.int32)[None]
        c.fill(rng, [(KINDS + 1) * ref.PAGE])
        self.kv = [c.rows(0, (KINDS + 1) * ref.PAGE, h) for h in range(kv_heads)]
        c.seqs, c.per_seq = len(hot_at), per
        self.table = rng.integers(0, KINDS, (len(hot_at), per)).astype(np.int32)
        self.table[np.arange(len(hot_at)), hot_at] = KINDS
        self.device = mmr.Kv8Pages(*c.upload(mmr).buffers[:4], ints(mmr, self.table), KINDS + 1, len(hot_at), per,
                                   kv_heads, D)

    def queries(self, rng, n, hq):
        group = hq // self.cache.kv_heads
        q = 0.3 * rng.standard_normal((n, hq, D))
        for h in range(hq):
            key = self.kv[h // group][0][KINDS * ref.PAGE + int(rng.integers(40))]
            q[:, h] += key * 20 * np.sqrt(D) / (key @ key)
        return q.reshape(n, -1).astype(np.float32)

    def expected(self, query, rows, context, hq):
        """As low_bit_reference.attention, whose bound this is too."""
        group = hq // self.cache.kv_heads
        out, bound = np.empty((len(query), hq, D)), np.empty((len(query), hq, D))
        for s in range(len(context)):
            for i in range(rows):
                keys = context[s] + i + 1
                full, rest = divmod(keys, ref.PAGE)
                times = np.repeat(np.bincount(self.table[s, :full], minlength=KINDS + 1), ref.PAGE).astype(np.float64)
                if rest:
                    times[self.table[s, full] * ref.PAGE:][:rest] += 1
                for h, (k, v) in enumerate(self.kv):
                    at = s * rows + i, slice(h * group, (h + 1) * group)
                    q = query[at[0]].reshape(hq, D)[at[1]].astype(np.float64)
                    score = q @ k.T / np.sqrt(D)
                    size = (np.abs(q) @ np.abs(k).T / np.sqrt(D)).max(-1) * 1.4427
                    p = times * np.exp(score - score.max(-1, keepdims=True))
                    out[at] = p @ v / p.sum(-1, keepdims=True)
                    steps = 8 * size + 2 + 16 * (keys // ref.PAGE + 1) + 32
                    bound[at] = (2 * steps * 2.0 ** -24)[:, None] * np.abs(v).max()
        return out.reshape(query.shape), bound.reshape(query.shape)


def check(mmr, hot_at, per, kv_heads, hq, rows):
    rng = np.random.default_rng(per + rows)
    r = Repeated(mmr, rng, hot_at, per, kv_heads)
    seqs = len(hot_at)
    context = [per * ref.PAGE - rows - 3 * (s % 5) for s in range(seqs)]
    query = r.queries(rng, seqs * rows, hq)
    got, error = attend(mmr, r.device, r.cache, query, np.arange(seqs + 1) * rows, context, hq, max_rows=rows)
    want, bound = r.expected(query, rows, context, hq)
    assert error == 0
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())
    # A weight is rounded to 2^-29 of about the largest, and the same pages again and again round to the same side: the
    # n keys of a row, whose weights sum to at least 1, together by up to n 2^-29 of |v|. Sums of P pages a wave are
    # off by P 2^-24, and the rest is as for shorter contexts.
    norm = np.linalg.norm(got - want) / np.linalg.norm(want)
    pages = per // 8 + 1
    size = np.abs(r.kv[0][1]).max() / np.sqrt((want ** 2).mean())
    assert norm <= per * ref.PAGE * 2.0 ** -29 * size + pages * 2.0 ** -24 + 4e-6, norm


# 256 blocks of a KV head and sequence each, which no split divides: eight waves take a page each in turn.
@pytest.mark.parametrize("per,hot_at", [
    (512, [0, 511, 504, 260]), (513, [512, 511, 504, 505]), (520, [512, 515, 519, 507]),
    (1032, [512, 1024, 1031, 519]), (8201, [8192, 8200, 4096, 519])])
def test_steps_of_many_pages_a_wave(gpu, per, hot_at):
    """64, 65, 129 and 1,026 pages a wave."""
    print(f"[case] {per} pages", flush=True)
    check(gpu, hot_at, per, 64, 64, 1)


@pytest.mark.parametrize("per,hot_at", [
    (512, [63, 64]), (520, [64, 65]), (520, [519, 454]), (1032, [64, 128]), (1032, [967, 1031])])
def test_many_rows_of_many_pages_a_split(gpu, per, hot_at):
    """Eight splits of 64, 65 and 129 pages: the 65th and 129th of a split are the first after a reading."""
    print(f"[case] {per} pages", flush=True)
    check(gpu, hot_at, per, 1, 8, 33)


def test_many_rows_of_many_pages_without_a_split(gpu):
    check(gpu, [64, 128, 129, 0, 63, 100, 65, 127, 126, 64] * 2, 130, 64, 64, 9)


# The second: added one by one, 33,408 keys a lane, each fp32 sum from 512 on would lose 0.45 of its step.
@pytest.mark.parametrize("weight", [2.0 ** -5, 2.0 ** -5 + 0.45 * 2.0 ** -14])
def test_sums_of_more_pages_than_an_int32_holds(gpu, weight):
    """Weights of 2^-5 are a digit of -128; with codes of 127, 64 of them a page, an int32 is full after 2,064 pages of
    a wave. One key of each wave outweighs the others 32 times and has the opposite value."""
    rng = np.random.default_rng(3)
    per, hkv, seqs = 16704, 64, 4  # 2,088 pages a wave
    r = Repeated(gpu, rng, [0] * seqs, per, hkv)
    c = r.cache
    r.table[:, :8] = KINDS  # the first page of each wave
    c.keys[:], c.values[:], c.key_exps[:], c.value_exps[:] = 0, 127, 0, 0
    c.keys[KINDS, :, 7, 0], c.values[KINDS, :, :, 7] = 64, -127
    device = gpu.Kv8Pages(*c.upload(gpu).buffers[:4], ints(gpu, r.table), KINDS + 1, seqs, per, hkv, D)
    query = np.zeros((seqs, hkv * D), np.float32)
    query[:, ::D] = -np.log(weight) * np.sqrt(D) / 64
    got, error = attend(gpu, device, c, query, np.arange(seqs + 1), [per * ref.PAGE - 1] * seqs, hkv, max_rows=1)
    others = (per * ref.PAGE - 8) * weight
    want = 127 * (others - 8) / (others + 8)
    assert error == 0
    # Sums of 2,088 pages a wave one after another, and 64 roundings of the rest.
    assert (np.abs(got - want) <= 2 * (2088 + 64) * 2.0 ** -24 * 127).all(), float(np.abs(got - want).max() / 127)
