"""Beams that only 64 bits tell apart, in both forms of the selection."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_beam_select import Select

pytestmark = pytest.mark.gpu


# Beams whose scores differ by less than 32 bits tell of their logarithms.  A row has n zeros among -inf: its terms and
# sum are whole numbers, so a token's score is s - log n, in 64 bits off by some 2^-49.  The scores are chosen so that
# two beams are 2^-42 to 2^-30 apart.
def close_pair(rng, vocab):
    while True:
        a, b = (int(n) for n in rng.integers(vocab // 2, vocab + 1, 2))
        exact = np.log(np.longdouble(a)) - np.log(np.longdouble(b))
        score = np.float32(exact)
        if abs(exact) < 2.0 ** -5 and 2.0 ** -42 < abs(np.longdouble(score) - exact) < 2.0 ** -30:
            return a, b, score, score > exact


@pytest.mark.parametrize("vocab", [2000, 6400, 40000])
def test_beams_apart_in_64_bits(gpu, vocab):
    mmr, rng, searches = gpu, np.random.default_rng(vocab), 150
    logits = np.full((2 * searches, vocab), -np.inf, np.float32)
    scores, best, tokens = np.zeros(2 * searches, np.float32), [], []
    for i in range(searches):
        *counts, scores[2 * i], first_wins = close_pair(rng, vocab)
        for r, n in zip((2 * i, 2 * i + 1), counts):
            logits[r, rng.permutation(vocab)[:n]] = 0.0
        best.append(2 * i + (0 if first_wins else 1))
        tokens.append(np.flatnonzero(logits[best[-1]] == 0)[:2])
    call = Select(mmr, logits, 2, -1, 0.0, scores, np.zeros(2 * searches, int), np.zeros(2 * searches, int))
    call.run()
    got = call.results()
    np.testing.assert_array_equal(got[3][: 2 * searches], np.repeat(best, 2))
    np.testing.assert_array_equal(got[4][: 2 * searches], np.concatenate(tokens))
