"""The 8-bit paged cache and 4-bit products in 64 bits, written from their definitions, for the tests."""
from __future__ import annotations

import numpy as np

PAGE, BLOCK = 64, 16


class Cache:
    """Host copy of an 8-bit paged cache."""

    def __init__(self, rng, pages, seqs, per_seq, kv_heads, d):
        # What a recycled page holds: any codes and any exponents.
        self.keys = rng.integers(-128, 128, (pages, kv_heads, PAGE, d)).astype(np.int8)
        self.values = rng.integers(-128, 128, (pages, kv_heads, d, PAGE)).astype(np.int8)
        self.key_exps = rng.integers(-128, 128, (pages, kv_heads, PAGE // BLOCK)).astype(np.int8)
        self.value_exps = rng.integers(-128, 128, (pages, kv_heads, PAGE // BLOCK)).astype(np.int8)
        assert pages >= seqs * per_seq
        self.table = rng.permutation(pages)[: seqs * per_seq].reshape(seqs, per_seq).astype(np.int32)
        self.pages, self.seqs, self.per_seq, self.kv_heads, self.d = pages, seqs, per_seq, kv_heads, d

    def upload(self, mmr):
        arrays = [mmr.DeviceArray.from_numpy(a)
                  for a in (self.keys, self.values, self.key_exps, self.value_exps, self.table)]
        return mmr.Kv8Pages(*arrays, self.pages, self.seqs, self.per_seq, self.kv_heads, self.d)

    def assert_equals(self, device):
        for name, buffer in zip(("keys", "values", "key_exps", "value_exps"), device.buffers):
            np.testing.assert_array_equal(buffer.numpy(), getattr(self, name), err_msg=name)

    def fill(self, rng, tokens, std=1.0, spread=0.3):
        """Cached tokens 0 .. tokens[s] - 1 of each sequence, of several sizes."""
        for s, n in enumerate(tokens):
            for t in range(0, n, BLOCK):
                page, block = self.table[s, t // PAGE], t % PAGE // BLOCK
                m = min(BLOCK, n - t)
                for codes, exps in ((self.keys, self.key_exps), (self.values.swapaxes(2, 3), self.value_exps)):
                    x = rng.standard_normal((self.kv_heads, m, self.d)) * std
                    x *= np.exp(spread * rng.standard_normal((self.kv_heads, 1, 1)))
                    for h in range(self.kv_heads):
                        e = exponent(np.abs(x[h]).max())
                        exps[page, h, block] = e
                        codes[page, h, t % PAGE: t % PAGE + m] = np.rint(x[h] * 2.0 ** -e)

    def rows(self, s, n, head):
        """Keys and values of the first n tokens of a sequence, [n][d] each."""
        pages = self.table[s, : -(-n // PAGE)]
        k = self.keys[pages, head].astype(np.float64)
        k *= np.repeat(2.0 ** self.key_exps[pages, head].astype(np.float64), BLOCK, -1)[..., None]
        v = self.values[pages, head].astype(np.float64).swapaxes(1, 2)
        v *= np.repeat(2.0 ** self.value_exps[pages, head].astype(np.float64), BLOCK, -1)[..., None]
        return k.reshape(-1, self.d)[:n], v.reshape(-1, self.d)[:n]


def exponent(top):
    if not top > 0:
        return -126
    e = int(np.ceil(np.log2(top / 127.0)))
    while top > 127.0 * 2.0 ** e:
        e += 1
    while top <= 127.0 * 2.0 ** (e - 1):
        e -= 1
    return min(max(e, -126), 122)


def normalised(x, w, eps):
    return x if w is None else x * w.astype(np.float64) / np.sqrt(np.mean(x * x, -1, keepdims=True) + float(np.float32(eps)))


def rotated(x, position, theta):
    d = x.shape[-1]
    # Angles in extended precision, whole turns taken off there.
    f = np.longdouble(theta) ** (-np.arange(0, d, 2).astype(np.longdouble) / d)
    tau = np.longdouble("6.283185307179586476925286766559005768")
    angle = np.longdouble(position) * f
    angle = (angle - np.rint(angle / tau) * tau).astype(np.float64)
    c, s = np.cos(angle), np.sin(angle)
    a, b = x[..., : d // 2], x[..., d // 2:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def append(cache, qkv, offsets, context, q_heads, theta, q_norm=None, k_norm=None, eps=1e-5, query=None):
    """Appends in place; returns the queries (rows outside the sequences as `query` has them)."""
    h, d = cache.kv_heads, cache.d
    x = qkv.astype(np.float64).reshape(len(qkv), q_heads + 2 * h, d)
    out = query.astype(np.float64).copy()
    for s in range(cache.seqs):
        n = offsets[s + 1] - offsets[s]
        blocks = {}
        for i in range(n):
            r, t = offsets[s] + i, context[s] + i
            with np.errstate(invalid="ignore", over="ignore"):
                out[r] = rotated(normalised(x[r, :q_heads], q_norm, eps), t, theta).reshape(-1)
                k = rotated(normalised(x[r, q_heads: q_heads + h], k_norm, eps), t, theta)
            blocks.setdefault(t // BLOCK, []).append((t, k, x[r, q_heads + h:]))
        for b, rows in blocks.items():
            page, block, first = cache.table[s, b * BLOCK // PAGE], b % (PAGE // BLOCK), rows[0][0]
            for which, codes, exps in ((1, cache.keys, cache.key_exps),
                                       (2, cache.values.swapaxes(2, 3), cache.value_exps)):
                for head in range(h):
                    new = np.stack([row[which][head] for row in rows])
                    finite = np.abs(new[np.isfinite(new)])
                    e = exponent(finite.max() if finite.size else 0.0)
                    if first % BLOCK:
                        held = int(exps[page, head, block])
                        old = slice(first // BLOCK * BLOCK % PAGE, first % PAGE)
                        if e > held:
                            codes[page, head, old] = np.rint(codes[page, head, old].astype(np.float64) * 2.0 ** (held - e))
                        e = max(e, held)
                    exps[page, head, block] = e
                    q = np.rint(np.nan_to_num(new * 2.0 ** -e, nan=0.0, posinf=np.inf, neginf=-np.inf))
                    codes[page, head, first % PAGE: first % PAGE + len(rows)] = np.clip(q, -127, 127)
    return out


def attention(cache, query, offsets, context, q_heads, out):
    """Rows in 64 bits (others as `out` has them), and a bound on what fp32 sums may be off by, row by row.

    A weight p = 2^s is off by the roundings of its score (q in fixed point, a sum and two products: 8 half steps of
    |s| and of the sum of |q k| that s may have cancelled), of the exponential (2), of a serial sum over at most
    every page's 16 keys a lane, and of the joins of waves and splits (32): relative to the weights' total, so the
    result is off by at most twice that of the largest |v|."""
    d, group = cache.d, q_heads // cache.kv_heads
    o, bound = out.astype(np.float64).copy(), np.zeros(out.shape)
    for s in range(cache.seqs):
        for i in range(offsets[s + 1] - offsets[s]):
            n, r = context[s] + i + 1, offsets[s] + i
            for head in range(q_heads):
                k, v = cache.rows(s, n, head // group)
                q = query[r, head * d:(head + 1) * d].astype(np.float64)
                score = k @ q / np.sqrt(d)
                size = (np.abs(k) @ np.abs(q) / np.sqrt(d)).max() * 1.4427
                p = np.exp(score - score.max())
                o[r, head * d:(head + 1) * d] = p @ v / p.sum()
                steps = 8 * size + 2 + 16 * (n // PAGE + 1) + 32
                bound[r, head * d:(head + 1) * d] = 2 * steps * 2.0 ** -24 * np.abs(v).max()
    return o, bound


def q4_weights(codes, scales, cols, group):
    """fp64 weights of packed codes: of 128 columns, word 4 p + j holds columns 32 j + 8 p + 0 .. 7."""
    c = np.arange(cols)
    byte = c // 128 * 64 + (c % 32 // 8 * 4 + c % 128 // 32) * 4 + c % 8 // 2
    n = (codes[:, byte].astype(np.int64) >> (c % 2 * 4)) & 15
    return np.where(n > 7, n - 16, n) * scales.astype(np.float64)[:, c // group]
