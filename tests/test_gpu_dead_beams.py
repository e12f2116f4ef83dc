"""Beam search whose masks leave fewer continuations than beams: steps with beams of no parent, which are empty
sequences until a later step gives them one again, over a decoder on the 8-bit paged cache, eagerly and from recorded
graphs."""
from __future__ import annotations

import numpy as np
import pytest

import low_bit_reference as ref
import paging_reference as paging
from test_gpu_beam_search import BEAMS, EOS, SHAPE, SINKS, VOCAB, WINDOW, View, WindowLayer
from test_gpu_beam_select import LSE
from test_gpu_low_bit_layer import EPS

pytestmark = pytest.mark.gpu


class Server:
    """Two searches over two layers; the calls of a step as they are documented."""

    def __init__(self, mmr, rng, prompts, recorded):
        self.mmr, self.prompts = mmr, prompts
        hidden, hq, hkv, d, ffn = SHAPE
        per, seqs, total = 4, len(prompts) * BEAMS, sum(prompts)
        up = mmr.DeviceArray.from_numpy

        def ints(values):
            return up(np.asarray(values, np.int32))

        def workspace(size):
            return mmr.DeviceArray(max(size, 1), np.uint8)

        self.ints, self.seqs, self.per = ints, seqs, per
        self.layers = [WindowLayer(mmr, hidden, hq, hkv, d, ffn, 64, total, rng) for _ in range(2)]
        self.layers[1].b["hidden"] = self.layers[0].b["out"]
        self.pool = paging.Pool(rng, 2, 24, seqs, per, hkv, d)
        self.refs, self.table, self.users = self.pool.upload(mmr)
        codes, scales = mmr.q4_quantize((rng.standard_normal((VOCAB, hidden)) * 0.12).astype(np.float32), 64)
        self.head, self.norm = (up(codes), up(scales)), up((1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32))
        self.embedding = up((rng.standard_normal((VOCAB, hidden)) * 0.8).astype(np.float16).view(np.uint16))
        self.logits = mmr.DeviceArray((seqs, VOCAB), np.float32)
        first = np.arange(len(prompts)) * BEAMS
        scores = np.full(seqs, -np.inf, np.float32)
        scores[first] = 0
        self.beams = mmr.Beams(up(scores), ints([0] * seqs), ints([0] * seqs))
        self.parent, self.token, self.keep, self.room = (ints([n] * seqs) for n in (-1, 0, 0, 0))
        self.offsets, self.context, self.error = ints(np.arange(seqs + 1)), ints([0] * seqs), ints([0])
        self.select_ws = workspace(mmr.beam_select_workspace_size(len(prompts), BEAMS, VOCAB))
        self.fork_ws = workspace(mmr.kv8_fork_workspace_size(seqs, per, self.pool.pages))
        self.attend_ws = workspace(max(mmr.kv8_window_attention_workspace_size(
            hq, hkv, d, seqs, n, most, per * 64, SINKS, WINDOW) for n, most in ((total, max(prompts)), (seqs, 1))))
        self.head_ws, self.stream = workspace(mmr.matvec_q4_workspace_size(hidden, seqs)), mmr.Stream()

        # Prompts: the first beam of a search brings its rows.
        rows = np.zeros(seqs, int)
        rows[first] = prompts
        self.room.upload(rows.astype(np.int32))
        self.fork()
        self.layers[0].b["hidden"].upload(rng.standard_normal((total, hidden)).astype(np.float32))
        offsets = np.concatenate([[0], np.cumsum(rows)])
        self.run_layers(total, max(prompts), ints(offsets))
        mmr.synchronize()
        self.check_fork([-1] * seqs, [0] * seqs, rows)
        self.check_layers(offsets, [0] * seqs, total)
        self.to_logits(up(np.repeat(self.layers[1].b["out"].numpy()[np.cumsum(prompts) - 1], BEAMS, 0)))
        self.room.upload(np.ones(seqs, np.int32))
        mmr.synchronize()
        self.select, self.go_on = self.run_select, self.run_step
        if recorded:
            graphs = []
            for run in (self.select, self.go_on):
                with mmr.Graph(self.stream) as graph:
                    run()
                graphs.append(graph)
            self.select, self.go_on = ((lambda graph=graph: graph.launch(self.stream)) for graph in graphs)

    def fork(self):
        self.mmr.kv8_fork(self.refs, self.users, self.parent, self.keep, self.room, self.fork_ws, self.error,
                          sinks=SINKS, window=WINDOW, stream=self.stream)

    def run_layers(self, n, most, offsets):
        for layer, pages in zip(self.layers, self.refs.layers):
            layer.run(pages, offsets, self.context, n, most, self.per * 64, self.attend_ws, self.stream)

    def to_logits(self, x):
        self.mmr.matvec_q4(*self.head, 64, VOCAB, SHAPE[0], x, self.seqs, self.logits, norm_w=self.norm, eps=EPS,
                           prologue=self.mmr.PRO_RMSNORM, workspace=self.head_ws, stream=self.stream)

    def run_select(self):
        self.mmr.beam_select(self.logits, len(self.prompts), BEAMS, VOCAB, EOS, 0.6, self.beams, self.beams,
                             self.parent, self.token, self.select_ws, self.error, stream=self.stream)

    def run_step(self):
        self.fork()
        self.mmr.embedding_gather(self.embedding, self.token, self.seqs, VOCAB, SHAPE[0], self.layers[0].b["hidden"],
                                  self.error, stream=self.stream)
        self.run_layers(self.seqs, 1, self.offsets)
        self.to_logits(self.layers[1].b["out"])

    def check_fork(self, *plan):
        assert paging.fork(self.pool, *plan, SINKS, WINDOW) == 0
        np.testing.assert_array_equal(self.table.numpy(), self.pool.table)
        np.testing.assert_array_equal(self.users.numpy(), self.pool.users)

    def check_layers(self, offsets, context, rows):
        for i, layer in enumerate(self.layers):
            layer.check(View(self.pool, i), offsets, context, rows)
        self.pool.assert_pages_equal()


@pytest.mark.parametrize("recorded", [False, True])
def test_masks_that_leave_fewer_continuations_than_beams(gpu, recorded):
    rng = np.random.default_rng(23)
    prompts = [120, 61]
    server = Server(gpu, rng, prompts, recorded)
    tokens = np.repeat(prompts, BEAMS) - 1  # of a row, after a step one more than of what it goes on from
    had_none = set()
    for i in range(12):
        x = server.logits.numpy()
        if i == 3:  # two continuations of the first search, both of its second beam
            x[0], x[2] = -np.inf, -np.inf
            x[1, np.argsort(x[1])[:-2]] = -np.inf
        if i == 6:  # one of the second, then one again
            x[4:] = -np.inf
        if i in (6, 7):
            x[3, np.arange(VOCAB) != 11] = -np.inf
        if i == 9:  # none of the first, which ends it
            x[:3] = -np.inf
        server.logits.upload(x)
        was = [b.numpy() for b in server.beams.buffers]
        server.select()
        gpu.synchronize()
        want, bits, gap = paging.select(x, BEAMS, EOS, 0.6, *was)
        assert bits == 0 and gap > LSE
        parent = server.parent.numpy()
        for got, w in zip([*server.beams.buffers[1:], server.parent, server.token], want[1:]):
            np.testing.assert_array_equal(got.numpy(), w)
        # A row without a parent has no tokens, whatever it had.
        tokens = np.where(parent < 0, 0, tokens[parent] + 1)
        server.keep.upload(tokens.astype(np.int32)), server.context.upload(tokens.astype(np.int32))
        server.go_on()
        gpu.synchronize()
        assert int(server.error.numpy()[0]) == 0
        server.check_fork(parent, tokens, [1] * server.seqs)
        server.check_layers(np.arange(server.seqs + 1), tokens, server.seqs)
        had_none |= {(i, int(r)) for r in np.flatnonzero(parent < 0)}
    assert had_none == {(3, 2), (6, 4), (6, 5), (7, 4), (7, 5)} | {(i, r) for i in (9, 10, 11) for r in range(3)}


def test_rows_without_a_parent_at_their_old_context(gpu):
    """Why: the pages of those places are gone, and the step is flagged."""
    server = Server(gpu, np.random.default_rng(23), [120, 61], False)
    x = server.logits.numpy()
    x[0, np.argsort(x[0])[:-2]] = -np.inf
    server.logits.upload(x)
    server.select()
    tokens = np.repeat([120, 61], BEAMS).astype(np.int32)
    server.keep.upload(tokens), server.context.upload(tokens)
    server.go_on()
    gpu.synchronize()
    np.testing.assert_array_equal(server.parent.numpy()[:3], [0, 0, -1])
    assert int(server.error.numpy()[0]) == 0  # nobody's tokens count as none
    assert all(int(layer.error.numpy()[0]) == paging.BAD_ROWS for layer in server.layers)
