"""Beam search of two searches over a small decoder on 4-bit weights and the 8-bit paged cache, as a server would run
it: prompts, then steps of selection, forking, layers with windowed attention and logits, eagerly and from a recorded
graph, and the pool compacted between.  Every call's result is checked on the inputs that the device had."""
from __future__ import annotations

import numpy as np
import pytest

import low_bit_reference as ref
import paging_reference as paging
from test_gpu_beam_select import LSE
from test_gpu_low_bit_layer import EPS, THETA, Layer
from test_gpu_q4 import product

pytestmark = pytest.mark.gpu
SHAPE = 256, 4, 2, 64, 512  # hidden, heads, KV heads, head dimension, FFN
VOCAB, BEAMS, SINKS, WINDOW = 601, 3, 4, 90
EOS = 7


class View:
    """One layer's pages of a pool, as low_bit_reference takes them."""

    def __init__(self, pool, layer):
        self.keys, self.values, self.key_exps, self.value_exps = (getattr(pool, n)[layer] for n in pool.NAMES)
        self.table, self.seqs, self.per_seq, self.kv_heads, self.d = (pool.table, pool.seqs, pool.per_seq,
                                                                      pool.kv_heads, pool.d)

    rows = ref.Cache.rows


class WindowLayer(Layer):
    def run(self, pages, offsets, context, rows, max_rows, max_tokens, workspace, stream=None):
        m, b = self.mmr, self.b
        self.matvec("qkv", "hidden", "qkv", rows, stream, norm_w=self.dnorms["input"], prologue=m.PRO_RMSNORM)
        m.kv8_append(b["qkv"], self.dnorms["q"], self.dnorms["k"], EPS, self.rope, pages, offsets, context, rows,
                     max_rows, self.hq, b["query"], self.error, stream=stream)
        m.kv8_window_attention(b["query"], pages, offsets, context, rows, max_rows, max_tokens, SINKS, WINDOW, self.hq,
                               b["attended"], workspace, self.error, stream=stream)
        self.matvec("o", "attended", "mid", rows, stream, residual=b["hidden"], epilogue=m.EPI_RESIDUAL)
        self.matvec("gate_up", "mid", "act", rows, stream, norm_w=self.dnorms["post"], prologue=m.PRO_RMSNORM,
                    epilogue=m.EPI_SWIGLU)
        self.matvec("down", "act", "out", rows, stream, residual=b["mid"], epilogue=m.EPI_RESIDUAL)

    def check(self, view, offsets, context, rows):
        got = {n: self.b[n].numpy()[:rows] for n in ("qkv", "query", "attended")}
        want = ref.append(view, got["qkv"], offsets, context, self.hq, THETA, self.norms["q"], self.norms["k"], EPS,
                          got["query"])
        assert (np.abs(got["query"] - want) <= 2.0 ** -24 * np.abs(want) + 1e-12).all()
        want, bound = paging.window_attention(view, got["query"], offsets, context, self.hq, SINKS, WINDOW,
                                              got["attended"])
        assert (np.abs(got["attended"] - want) <= bound).all()
        assert int(self.error.numpy()[0]) == 0


@pytest.mark.parametrize("recorded", [False, True])
def test_search(gpu, recorded):
    mmr, rng = gpu, np.random.default_rng(17)
    hidden, hq, hkv, d, ffn = SHAPE
    prompts, steps, per = [120, 61], 14, 4
    seqs, total = len(prompts) * BEAMS, sum(prompts)
    first = np.arange(len(prompts)) * BEAMS  # the row of a search's first beam
    up = mmr.DeviceArray.from_numpy

    def ints(values):
        return up(np.asarray(values, np.int32))

    layers = [WindowLayer(mmr, hidden, hq, hkv, d, ffn, 64, total, rng) for _ in range(2)]
    layers[1].b["hidden"] = layers[0].b["out"]
    pool = paging.Pool(rng, 2, 24, seqs, per, hkv, d)
    refs, table, users = pool.upload(mmr)
    codes, scales = mmr.q4_quantize((rng.standard_normal((VOCAB, hidden)) * 0.12).astype(np.float32), 64)
    head, exact_head = (up(codes), up(scales)), ref.q4_weights(codes, scales, hidden, 64)
    norm = (1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32)
    embedding = (rng.standard_normal((VOCAB, hidden)) * 0.8).astype(np.float16)
    d_embedding, d_norm = up(embedding.view(np.uint16)), up(norm)
    logits = mmr.DeviceArray((seqs, VOCAB), np.float32)
    scores = np.full(seqs, -np.inf, np.float32)
    scores[first] = 0
    beams = mmr.Beams(up(scores), ints([0] * seqs), ints([0] * seqs))
    parent, token, keep, room = ints([-1] * seqs), ints([0] * seqs), ints([0] * seqs), ints([0] * seqs)
    offsets, context, error = ints(np.arange(seqs + 1)), ints([0] * seqs), ints([0])

    def workspace(size):
        return mmr.DeviceArray(max(size, 1), np.uint8)

    select_ws = workspace(mmr.beam_select_workspace_size(len(prompts), BEAMS, VOCAB))
    fork_ws = workspace(mmr.kv8_fork_workspace_size(seqs, per, pool.pages))
    attend_ws = workspace(max(mmr.kv8_window_attention_workspace_size(hq, hkv, d, seqs, n, most, per * 64, SINKS, WINDOW)
                              for n, most in ((total, max(prompts)), (seqs, 1))))
    head_ws = workspace(mmr.matvec_q4_workspace_size(hidden, seqs))
    stream = mmr.Stream()

    def fork():
        mmr.kv8_fork(refs, users, parent, keep, room, fork_ws, error, sinks=SINKS, window=WINDOW, stream=stream)

    def run_layers(n, most, d_offsets):
        for layer, pages in zip(layers, refs.layers):
            layer.run(pages, d_offsets, context, n, most, per * 64, attend_ws, stream)

    def to_logits(x):
        mmr.matvec_q4(*head, 64, VOCAB, hidden, x, seqs, logits, norm_w=d_norm, eps=EPS, prologue=mmr.PRO_RMSNORM,
                      workspace=head_ws, stream=stream)

    def step():
        mmr.beam_select(logits, len(prompts), BEAMS, VOCAB, EOS, 0.6, beams, beams, parent, token, select_ws, error,
                        stream=stream)
        fork()
        mmr.embedding_gather(d_embedding, token, seqs, VOCAB, hidden, layers[0].b["hidden"], error, stream=stream)
        run_layers(seqs, 1, offsets)
        to_logits(layers[1].b["out"])

    def check_fork(plan):
        assert paging.fork(pool, *plan, SINKS, WINDOW) == 0
        np.testing.assert_array_equal(table.numpy(), pool.table)
        np.testing.assert_array_equal(users.numpy(), pool.users)

    # Prompts: the first beam of a search brings its rows, the others none.
    rows = np.zeros(seqs, int)
    rows[first] = prompts
    room.upload(rows.astype(np.int32))
    fork()
    layers[0].b["hidden"].upload(rng.standard_normal((total, hidden)).astype(np.float32))
    prompt_offsets = np.concatenate([[0], np.cumsum(rows)])
    run_layers(total, max(prompts), ints(prompt_offsets))
    mmr.synchronize()
    check_fork(([-1] * seqs, [0] * seqs, rows))
    for i, layer in enumerate(layers):
        layer.check(View(pool, i), prompt_offsets, [0] * seqs, total)
    pool.assert_pages_equal()
    ends = np.repeat(layers[1].b["out"].numpy()[np.cumsum(prompts) - 1], BEAMS, 0)
    last = up(ends)
    to_logits(last)
    tokens = np.repeat(prompts, BEAMS)
    room.upload(np.ones(seqs, np.int32))
    mmr.synchronize()
    want, off = product(exact_head, ends, norm, 1, EPS, mmr.EPI_STORE, None, mmr)
    assert (np.abs(logits.numpy() - want) <= off).all()

    if recorded:
        with mmr.Graph(stream) as graph:
            step()
    history, ended_once = [], False
    for i in range(steps):
        was = [b.numpy() for b in beams.buffers]
        x = logits.numpy()
        # Every beam of a search has the parent's first tokens; the others of the first step hold nothing to keep.
        keep.upload(tokens.astype(np.int32)), context.upload(tokens.astype(np.int32))
        if recorded:
            graph.launch(stream)
        else:
            step()
        mmr.synchronize()
        assert int(error.numpy()[0]) == 0
        want, bits, gap = paging.select(x, BEAMS, EOS, 0.6, *was)
        assert bits == 0 and gap > LSE
        got = [b.numpy() for b in beams.buffers] + [parent.numpy(), token.numpy()]
        for g, w in zip(got[1:], want[1:]):
            np.testing.assert_array_equal(g, w)
        assert (np.abs(got[0] - want[0]) <= LSE + 2.0 ** -24 * np.abs(want[0])).all()
        check_fork((got[3], tokens, [1] * seqs))
        np.testing.assert_array_equal(layers[0].b["hidden"].numpy()[:seqs], embedding[got[4]].astype(np.float32))
        for n, layer in enumerate(layers):
            layer.check(View(pool, n), np.arange(seqs + 1), tokens, seqs)
        pool.assert_pages_equal()
        assert (pool.users[pool.table[np.arange(seqs), tokens // 64]] == 1).all()
        tokens = tokens + 1
        history.append((got[3], got[4]))
        ended_once = ended_once or got[2].any()
        if i == steps // 2:
            moved, live = ints(np.zeros(pool.pages)), ints([0])
            mmr.kv8_compact(refs, users, table, users, moved, live, workspace(mmr.kv8_compact_workspace_size(pool.pages)),
                            stream=stream)
            mmr.synchronize()
            want_moved, want_live = paging.compact(pool)
            np.testing.assert_array_equal(table.numpy(), pool.table)
            np.testing.assert_array_equal(moved.numpy(), want_moved)
            assert int(live.numpy()[0]) == want_live
            pool.assert_pages_equal()
    # The windows of both searches have left their second page behind, or will before long; the first has sinks.
    assert (pool.table[:, 0] >= 0).all()
    # Beams of one search are of one search, and no two of them the same.
    for f in first:
        paths = set()
        for b in range(f, f + BEAMS):
            path, at = [], b
            for p, t in reversed(history):
                path.append(int(t[at]))
                at = p[at]
            assert at in range(f, f + BEAMS)
            paths.add(tuple(path))
        assert len(paths) == BEAMS
