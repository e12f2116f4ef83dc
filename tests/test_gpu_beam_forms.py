"""Beam selection where rows are several runs, which a second kernel joins: masks,
values that are not finite and ended beams."""
from __future__ import annotations

import numpy as np
import pytest

import paging_reference as paging
from test_gpu_beam_select import LOWEST, Select, beams_of, logits_of

pytestmark = pytest.mark.gpu


def select(mmr, logits, beams, *rest, fill=0xFF):
    """A call that needs a workspace, and so has the two kernels; of the workspace every byte is `fill`."""
    call = Select(mmr, logits, beams, *rest)
    assert call.workspace.nbytes > 0
    call.workspace.upload(np.full(call.workspace.nbytes, fill, np.uint8))
    call.run()
    return call


# Scores are checked with the bound of test_gpu_beam_select, whose entropy of 11.5 holds here, too: the logits'
# exponentials are far from alike (0.7 in a row of 300,001).
# Some of a row's runs of 4,096 columns are masked as a whole, with few tokens left.
@pytest.mark.parametrize("mask", [-np.inf, LOWEST, -1e30])
@pytest.mark.parametrize("left", [0, 1, 3, 40])
@pytest.mark.parametrize("searches,beams,vocab", [(2, 5, 20000), (1, 32, 6400), (2, 3, 300001)])
def test_masked_logits_of_several_runs(gpu, searches, beams, vocab, left, mask):
    print(f"[case] masked {searches},{beams},{vocab} left {left} mask {mask}", flush=True)
    rng = np.random.default_rng(left + vocab)
    rows = searches * beams
    logits = logits_of(rng, rows, vocab)
    for r in range(rows):
        if r % 2 == 0 or left == 0:
            logits[r, rng.permutation(vocab)[left:]] = mask
    call = select(gpu, logits, beams, 2, 0.0, -np.arange(float(rows)) * 0.37, np.arange(rows), np.zeros(rows, int))
    assert call.check() == 0


@pytest.mark.parametrize("beams,vocab", [(4, 20000), (16, 6400), (4, 300001)])
def test_what_is_not_finite_in_several_runs(gpu, beams, vocab):
    """In a row's first run, in a later one, in one of more than 64, in a whole run; scores; an ended beam's logits."""
    rng = np.random.default_rng(vocab)
    rows = 4 * beams
    logits = logits_of(rng, rows, vocab)
    logits[1, vocab - 10], logits[beams, 0], logits[beams + 1, 5000] = np.nan, np.inf, np.inf
    logits[beams + 2, 4096:] = -np.inf  # all but the first run
    logits[2 * beams, 4096:8192], logits[2 * beams + 1, :4096] = np.nan, -np.inf
    scores, lengths, ended = beams_of(rng, rows, 0.0)
    scores[3 * beams: 3 * beams + 3] = np.nan, np.inf, -np.inf
    logits[3 * beams + 2, 7] = np.nan  # of a beam that has no candidates anyway
    logits[3 * beams + 3], ended[3 * beams + 3] = np.nan, True
    call = select(gpu, logits, beams, 2, 0.0, scores, lengths, ended)
    assert call.check() == paging.NOT_FINITE
    # Without those of the logits and scores, the ended beam's logits are not read.
    for r in (1, beams, beams + 1, 2 * beams, 3 * beams + 2):
        logits[r] = logits[beams + 3]
    scores[3 * beams: 3 * beams + 2] = -3.5, -4.25
    assert select(gpu, logits, beams, 2, 0.0, scores, lengths, ended).check() == 0
    # A search of which nothing is left, beside those that are in order.
    logits[:beams, 4097] = np.nan
    call = select(gpu, logits, beams, 2, 0.0, scores, lengths, ended)
    assert call.check() == paging.NOT_FINITE
    assert (call.results()[3][:beams] == -1).all()


@pytest.mark.parametrize("fill", [0x00, 0xFF, 0x3F])
@pytest.mark.parametrize("ended", [[1, 1, 1, 1], [1, 0, 0, 1], [0, 0, 1, 0]])
def test_ended_beams_of_several_runs(gpu, ended, fill):
    """What an ended beam has in the workspace is never written, and never used."""
    rng = np.random.default_rng(3)
    for vocab in (20000, 300001):
        logits = logits_of(rng, 4, vocab)
        logits[np.flatnonzero(ended)] = np.nan
        rest = [-3.0, -4.0, -50.0, -6.0], [3, 4, 5, 6], ended
        assert select(gpu, logits, 4, 5, 1.0, *rest, fill=fill).check() == 0
        logits[np.flatnonzero(ended)] = 0.5
        call = select(gpu, logits, 4, -1, 1.0, *rest, fill=fill)  # without an end token the flags say nothing
        assert call.check() == 0 and (call.results()[2][:4] == 0).all()


@pytest.mark.parametrize("vocab", [9000, 20000, 300001])
def test_first_step_of_several_runs(gpu, vocab):
    rng = np.random.default_rng(vocab)
    logits = logits_of(rng, 8, vocab)
    scores = np.array([0, -np.inf, -np.inf, -np.inf] * 2, np.float32)
    assert select(gpu, logits, 4, -1, 0.0, scores, np.zeros(8, int), np.ones(8, int)).check() == 0
    # One token is left of the one beam: the others of its search have no parent.
    logits[0, np.arange(vocab) != vocab - 2] = -np.inf
    call = select(gpu, logits, 4, 3, 0.0, scores, np.zeros(8, int), np.zeros(8, int))
    assert call.check() == 0
    np.testing.assert_array_equal(call.results()[3][:4], [0, -1, -1, -1])
    np.testing.assert_array_equal(call.results()[4][:4], [vocab - 2, 3, 3, 3])
