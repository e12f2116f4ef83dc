"""The best continuations of beams against 64 bits: parents, tokens and lengths exactly, scores to the roundings of
their sums."""
from __future__ import annotations

import numpy as np
import pytest

import paging_reference as paging

pytestmark = pytest.mark.gpu

# A log of a sum of exponentials is off by the relative error of the sum, in half steps: two of each term's exponent
# (a difference and a product) times that exponent, in the mean over the terms, which is at most the entropy, so the log
# of the number of terms (11.5 for 100,000); the exponentials of a term and of what brings the sums of a wave and of a
# run to one reference (2 each); sums of 16 terms and of their halves (17), of 64 lanes (6), of four waves (3); and the
# logarithm (2): 23 + 6 + 26 + 2 = 57.
LSE = 2.0 ** -24 * 57


class Select:
    def __init__(self, mmr, logits, beams, eos, power, scores, lengths, ended, extra=2):
        scores, lengths, ended = np.asarray(scores, np.float32), np.asarray(lengths), np.asarray(ended)
        self.mmr, self.case = mmr, (logits, beams, eos, power, scores, lengths, ended)
        rows, vocab = logits.shape
        self.searches, self.beams, self.vocab, self.eos, self.power = rows // beams, beams, vocab, eos, power
        up = mmr.DeviceArray.from_numpy
        self.logits = up(logits)
        self.before = mmr.Beams(up(np.asarray(scores, np.float32)), up(np.asarray(lengths, np.int32)),
                                up(np.asarray(ended, np.int32)))
        # Rows behind the last beam stay as they are.
        self.after = mmr.Beams(up(np.full(rows + extra, 7.5, np.float32)), up(np.full(rows + extra, 77, np.int32)),
                               up(np.full(rows + extra, 77, np.int32)))
        self.parent, self.token = (up(np.full(rows + extra, 77, np.int32)) for _ in range(2))
        self.error = up(np.zeros(1, np.int32))
        size = mmr.beam_select_workspace_size(self.searches, beams, vocab)
        self.workspace = up(np.full(size, 0xFF, np.uint8))

    def run(self, after=None, stream=None, workspace=None):
        self.mmr.beam_select(self.logits, self.searches, self.beams, self.vocab, self.eos, self.power, self.before,
                             after or self.after, self.parent, self.token, workspace or self.workspace, self.error,
                             stream=stream)

    def results(self, after=None):
        return [b.numpy() for b in (*(after or self.after).buffers, self.parent, self.token)]

    def check(self, after=None):
        rows = self.searches * self.beams
        want, error, gap = paging.select(*self.case)
        assert gap > LSE  # what is next to each other is told apart by sums that are off by so much
        got = self.results(after)
        for name, g, w in zip(("lengths", "ended", "parent", "token"), got[1:], want[1:]):
            np.testing.assert_array_equal(g[:rows], w, err_msg=name)
        none = want[3] < 0
        assert (got[0][:rows][none] == -np.inf).all()
        off = np.abs(got[0][:rows][~none].astype(np.float64) - want[0][~none])
        assert (off <= LSE + 2.0 ** -24 * np.abs(want[0][~none])).all(), off.max()
        for g in got:
            assert (g[rows:] == (7.5 if g.dtype == np.float32 else 77)).all()
        assert int(self.error.numpy()[0]) == error
        return error


def beams_of(rng, rows, done=0.2):
    lengths = rng.integers(0, 40, rows)
    return (-2.0 * lengths * np.exp(0.2 * rng.standard_normal(rows))).astype(np.float32), lengths, rng.random(rows) < done


def logits_of(rng, rows, vocab):
    return (2 * rng.standard_normal((rows, vocab)) + 3 * np.exp(0.6 * rng.standard_normal((rows, vocab)))).astype(np.float32)


SIZES = [(1, 1, 1), (1, 4, 6400), (3, 5, 257), (2, 32, 33), (1, 32, 5), (2, 32, 1), (2, 8, 100003), (1, 3, 4096),
         (1, 3, 4097), (4, 16, 12289), (1, 1, 6400), (5, 2, 63), (1, 32, 20000), (300, 2, 700), (2, 7, 16385),
         (1, 2, 1023), (1, 2, 1025),
         # On both sides of what one block takes: 16 waves of 2,048 columns each.
         (2, 16, 2048), (2, 16, 2049), (1, 8, 4096), (1, 8, 4097), (3, 5, 6144), (3, 5, 6145), (2, 4, 8192), (1, 4, 8193),
         (2, 1, 32768), (1, 1, 32769), (1, 16, 6400), (1, 31, 6400), (1, 16, 100)]


@pytest.mark.parametrize("searches,beams,vocab", SIZES)
@pytest.mark.parametrize("power", [0.0, 0.6, 2.0])
def test_select(gpu, searches, beams, vocab, power):
    print(f"[case] select {searches},{beams},{vocab} power {power}", flush=True)
    rng = np.random.default_rng(vocab + beams)
    rows = searches * beams
    call = Select(gpu, logits_of(rng, rows, vocab), beams, min(2, vocab - 1), power, *beams_of(rng, rows))
    call.run()
    call.check()


@pytest.mark.parametrize("vocab", [3, 4, 5, 700, 6400, 9001])
def test_first_step(gpu, vocab):
    """One beam of score 0 and the others at -inf, whose logits are anything."""
    rng = np.random.default_rng(vocab)
    logits = logits_of(rng, 8, vocab)
    scores = np.array([0, -np.inf, -np.inf, -np.inf] * 2, np.float32)
    call = Select(gpu, logits, 4, -1, 0.0, scores, np.zeros(8, int), np.ones(8, int))
    call.run()
    assert call.check() == 0
    if vocab == 3:
        assert call.results()[3][3] == -1


def test_ended_beams_stay(gpu):
    rng = np.random.default_rng(3)
    for ended in ([1, 1, 1, 1], [1, 0, 0, 1], [0, 0, 1, 0]):
        logits = logits_of(rng, 4, 3000)
        logits[np.flatnonzero(ended)] = np.nan  # not read
        call = Select(gpu, logits, 4, 5, 1.0, [-3.0, -4.0, -50.0, -6.0], [3, 4, 5, 6], ended)
        call.run()
        assert call.check() == 0
    # Without an end token the flags say nothing.
    call = Select(gpu, logits_of(rng, 4, 3000), 4, -1, 1.0, [-3.0, -4.0, -50.0, -6.0], [3, 4, 5, 6], [1, 1, 1, 1])
    call.run()
    assert call.check() == 0 and (call.results()[2][:4] == 0).all()


LOWEST = float(np.finfo(np.float32).min)


@pytest.mark.parametrize("mask", [-np.inf, LOWEST, -1e30])
@pytest.mark.parametrize("left", [0, 1, 3, 40])
def test_masked_logits(gpu, mask, left):
    """Rows of which little or nothing is left; masks of the type's lowest value are candidates behind all others."""
    rng = np.random.default_rng(left)
    logits = logits_of(rng, 10, 5000)
    for r in range(10):
        if r % 2 == 0 or left == 0:
            logits[r, rng.permutation(5000)[left:]] = mask
    call = Select(gpu, logits, 5, 2, 0.0, -np.arange(10.0) * 0.37, np.arange(10), np.zeros(10, int))
    call.run()
    assert call.check() == 0


def test_what_is_not_finite(gpu):
    rng = np.random.default_rng(4)
    logits = logits_of(rng, 12, 4500)
    logits[1, 4400], logits[5, 0], logits[6, 3] = np.nan, np.inf, -np.inf
    scores, lengths, ended = beams_of(rng, 12, 0.0)
    scores[8], scores[9], scores[10] = np.nan, np.inf, -np.inf
    call = Select(gpu, logits, 4, 2, 0.0, scores, lengths, ended)
    call.run()
    assert call.check() == paging.NOT_FINITE
    # A search of which nothing is left, beside one that is in order.
    logits = logits_of(rng, 4, 4500)
    logits[:2, 7] = np.nan
    call = Select(gpu, logits, 2, 2, 0.0, [-1.0, -2.0, -1.0, -2.0], [1, 1, 1, 1], [0, 0, 0, 0])
    call.run()
    assert call.check() == paging.NOT_FINITE
    assert (call.results()[3][:2] == -1).all() and (call.results()[3][2:4] >= 2).all()


@pytest.mark.parametrize("vocab", [40, 300, 4096, 6400, 20481])
@pytest.mark.parametrize("beams", [1, 8, 32])
def test_equal_values(gpu, vocab, beams):
    """All logits alike, few different ones, rows that are the same: the lower beam, then the lower token."""
    rng = np.random.default_rng(vocab)
    scores = np.full(beams, -1.5, np.float32)
    one = rng.integers(0, 3, vocab)
    for logits in (np.zeros((beams, vocab)), rng.integers(0, 3, (beams, vocab)), np.tile(one, (beams, 1)),
                   np.tile(logits_of(rng, 1, vocab), (beams, 1))):
        call = Select(gpu, logits.astype(np.float32), beams, -1, 0.6, scores, np.full(beams, 3), np.zeros(beams, int))
        call.run()
        call.check()


def test_in_place_and_always_the_same(gpu):
    mmr, rng = gpu, np.random.default_rng(6)
    for searches, beams, vocab in ((3, 4, 6400), (2, 32, 9000), (5, 1, 100)):
        rows = searches * beams
        call = Select(mmr, logits_of(rng, rows, vocab), beams, 2, 0.6, *beams_of(rng, rows))
        call.run()
        call.check()
        want = [g[:rows] for g in call.results()]
        before = [b.numpy() for b in call.before.buffers]
        for _ in range(10):
            for b, a in zip(call.before.buffers, before):
                b.upload(a)
            call.run(after=call.before)
            for g, w in zip(call.results(call.before), want):
                np.testing.assert_array_equal(g[:rows], w)


def test_largest_sizes(gpu):
    """Tokens of 24 bits, and as many searches as there may be."""
    rng = np.random.default_rng(9)
    logits = rng.standard_normal((2, 1 << 24)).astype(np.float32)
    logits[0, [(1 << 24) - 1, 5]], logits[1, [0, (1 << 24) - 2]] = [9.0, 8.5], [8.75, 9.25]
    call = Select(gpu, logits, 2, (1 << 24) - 1, 0.6, [-3.0, -2.5], [4, 4], [0, 0])
    call.run()
    call.check()
    logits = rng.standard_normal((65535, 3)).astype(np.float32)
    call = Select(gpu, logits, 1, 1, 1.0, *beams_of(rng, 65535))
    call.run()
    call.check()


def test_searches_on_two_streams(gpu):
    mmr, rng = gpu, np.random.default_rng(10)
    streams, calls = [mmr.Stream(), mmr.Stream()], []
    for searches, beams, vocab in ((40, 4, 6400), (20, 8, 30000)):
        calls.append(Select(mmr, logits_of(rng, searches * beams, vocab), beams, 2, 0.6, *beams_of(rng, searches * beams)))
    mmr.synchronize()
    for _ in range(20):
        for call, stream in zip(calls, streams):
            call.run(stream=stream)
    mmr.synchronize()
    for call in calls:
        call.check()


def test_recorded_calls_share_a_workspace(gpu):
    mmr, rng, stream = gpu, np.random.default_rng(7), gpu.Stream()
    calls = []
    for searches, beams, vocab in ((1, 4, 6400), (6, 5, 4097), (2, 2, 30000)):
        rows = searches * beams
        calls.append(Select(mmr, logits_of(rng, rows, vocab), beams, 2, 0.6, *beams_of(rng, rows)))
    workspace = max((c.workspace for c in calls), key=lambda w: w.nbytes)
    graphs = []
    for c in calls:
        with mmr.Graph(stream) as graph:
            c.run(stream=stream, workspace=workspace)
        graphs.append(graph)
    for order in ([0, 1, 2], [2, 1, 0], [1, 1, 0, 2], [0, 2, 0, 1]):
        for c in calls:
            for b in (*c.after.buffers, c.parent, c.token):
                b.upload(np.full(b.shape, 7.5 if b.dtype == np.float32 else 77, b.dtype))
        mmr.synchronize()
        for i in order:
            graphs[i].launch(stream)
        calls[order[0]].run(stream=stream, workspace=workspace)
        mmr.synchronize()
        for c in calls:
            c.check()


def test_logits_past_eight_gigabytes(gpu):
    """Rows whose first logit has an offset of more than 31 bits: the last search differs from the others."""
    mmr, rng = gpu, np.random.default_rng(8)
    beams, vocab = 2, 100003
    searches = 2 ** 31 // vocab // beams + 2
    rows = searches * beams
    logits = mmr.DeviceArray((rows, vocab), np.float32, zero=True)
    last = logits_of(rng, beams, vocab)
    mmr.check(mmr.lib().mmr_memcpy_h2d(logits.ptr + (rows - beams) * vocab * 4, last.ctypes.data, last.nbytes))
    scores, lengths, ended = np.tile([-1.0, -2.0], searches).astype(np.float32), np.ones(rows, int), np.zeros(rows, int)
    call = Select(mmr, np.zeros((beams, vocab), np.float32), beams, -1, 0.0, scores, lengths, ended)
    call.searches, call.logits = searches, logits
    call.after = mmr.Beams(*(mmr.DeviceArray(rows, t) for t in (np.float32, np.int32, np.int32)))
    call.parent, call.token = (mmr.DeviceArray(rows, np.int32) for _ in range(2))
    call.workspace = mmr.DeviceArray(mmr.beam_select_workspace_size(searches, beams, vocab), np.uint8)
    call.run()
    got = call.results()
    # Of equal logits the first tokens of the better beam.
    np.testing.assert_array_equal(got[3][:-2], np.repeat(np.arange(searches - 1) * 2, 2))
    np.testing.assert_array_equal(got[4][:-2], np.tile([0, 1], searches - 1))
    want, _, gap = paging.select(last, beams, -1, 0.0, scores[:2], lengths[:2], ended[:2])
    assert gap > LSE
    np.testing.assert_array_equal(got[3][-2:], want[3] + rows - 2)
    np.testing.assert_array_equal(got[4][-2:], want[4])
