"""Host side of the window, the pages and the beams: sizes and refusals (no GPU needed: every refusal comes before any
launch), and the references of the GPU tests against brute force."""
from __future__ import annotations

import numpy as np
import pytest

import low_bit_reference as ref
import paging_reference as paging
from test_low_bit_cpu import BAD_PAGES, At, pages


def refuser(mmr, call, good):
    def refused(message, **change):
        with pytest.raises(mmr.InvalidArgument, match=message):
            call(**{**good, **change})

    return refused


def test_window_attention_refuses(mmr):
    b = At()
    good = dict(query=b, cache=pages(mmr), offsets=b, context=b, rows=4, max_rows=1, max_tokens=200, sinks=4,
                window=100, q_heads=8, out=b, workspace=b, error=b)
    refused = refuser(mmr, mmr.kv8_window_attention, good)
    for name in ("query", "offsets", "context", "out", "error"):
        refused("null", **{name: At(None)})
    refused("window", window=0)
    refused("window", window=-1)
    refused("sinks", sinks=-1)
    refused("aligned", query=At(4100))
    refused("max_rows", max_rows=5)
    refused("max_tokens", max_tokens=257)
    refused("q_heads", q_heads=3)
    need = mmr.kv8_window_attention_workspace_size(8, 2, 96, 1, 1, 1, 1 << 18, 64, 1 << 17)
    assert need > 0
    big = dict(cache=pages(mmr, seqs=1, pages_per_seq=4096), rows=1, max_tokens=1 << 18, sinks=64, window=1 << 17)
    refused("null workspace", **big, workspace=None)
    refused("too small", **big, workspace=At(4096, need - 1))
    for message, change in BAD_PAGES:
        refused(message, cache=pages(mmr, **change))


def test_window_attention_workspace(mmr):
    def size(sinks, window, max_tokens=1 << 15, rows=1):
        return mmr.kv8_window_attention_workspace_size(8, 2, 96, 1, rows, rows, max_tokens, sinks, window)

    whole = mmr.kv8_attention_workspace_size(8, 2, 96, 1, 1, 1, 1 << 15)
    # Windows of all keys are the call without one; short ones need no split.
    assert size(0, 1 << 15) == size(0, 1 << 40) == size(1 << 15, 1) == size(1 << 62, 1) == whole > 0
    assert size(4, 500) == 0
    assert 0 < size(4, 1 << 13) <= whole
    assert size(0, (1 << 15) - 1) > 0
    for sinks, window in ((-1, 5), (0, 0), (0, -1), (-(1 << 62), 1)):
        assert size(sinks, window) == 0
    assert size(4, 5000, 0) == size(4, 5000, -1) == size(4, 5000, 1 << 62) == 0


def layers(mmr, count=2, **change):
    return mmr.Kv8Layers(pages(mmr, **change) for _ in range(count))


def test_fork_refuses(mmr):
    b = At()
    good = dict(layers=layers(mmr), users=b, parent=b, keep=b, room=b, workspace=b, error=b)
    refused = refuser(mmr, mmr.kv8_fork, good)
    for name in ("users", "parent", "keep", "room", "error"):
        refused("null", **{name: At(None)})
    refused("null workspace", workspace=At(None))
    refused("aligned", users=At(4100))
    refused("aligned", workspace=At(4104))
    refused("sinks", sinks=-1)
    refused("sinks", window=-1)
    need = mmr.kv8_fork_workspace_size(2, 4, 10)
    assert need > 0
    refused("too small", workspace=At(4096, need - 1))
    refused("layers", layers=layers(mmr, 0))
    refused("layers", layers=layers(mmr, 4097))
    for message, change in BAD_PAGES:
        if message != "q_heads":
            refused(message, layers=layers(mmr, **change))
    refused("2\\^24", layers=layers(mmr, pages=(1 << 24) + 1))
    refused("2\\^28", layers=layers(mmr, seqs=65535, pages_per_seq=1 << 14))
    for change in (dict(pages=11), dict(seqs=3), dict(pages_per_seq=5), dict(kv_heads=1), dict(head_dim=64),
                   dict(table=At(8192))):
        refused("one shape", layers=mmr.Kv8Layers([pages(mmr), pages(mmr, **change)]))
    with pytest.raises(mmr.InvalidArgument, match="null layers"):
        mmr.check(mmr.lib().mmr_kv8_fork(None, 1, 4096, 4096, 4096, 4096, 0, 0, 4096, 1 << 20, 4096, None))


def test_compact_refuses(mmr):
    b = At()
    good = dict(layers=layers(mmr), users=b, table_out=b, users_out=b, moved=b, live=b, workspace=b)
    refused = refuser(mmr, mmr.kv8_compact, good)
    for name in ("users", "table_out", "users_out", "moved", "live"):
        refused("null", **{name: At(None)})
    refused("null workspace", workspace=At(None))
    for name in ("users", "users_out", "moved", "workspace"):
        refused("aligned", **{name: At(4100)})
    refused("too small", workspace=At(4096, mmr.kv8_compact_workspace_size(10) - 1))
    refused("2\\^24", layers=layers(mmr, pages=(1 << 24) + 1))


def test_select_refuses(mmr):
    b = At()
    beams = mmr.Beams(b, b, b)
    good = dict(logits=b, searches=2, beams=4, vocab=50000, eos=2, length_power=0.5, before=beams, after=beams, parent=b,
                token=b, workspace=b, error=b)
    refused = refuser(mmr, mmr.beam_select, good)
    for name in ("logits", "parent", "token", "error"):
        refused("null", **{name: At(None)})
    for name in ("before", "after"):
        for i in range(3):
            parts = [b, b, b]
            parts[i] = At(None)
            refused("null beams", **{name: mmr.Beams(*parts)})
    refused("null workspace", workspace=At(None))
    refused("aligned", logits=At(4100))
    refused("aligned", workspace=At(4104))
    refused("searches", searches=0)
    refused("searches", searches=65536)
    refused("beams", beams=0)
    refused("beams", beams=33)
    refused("vocab", vocab=0)
    refused("vocab", vocab=(1 << 24) + 1)
    refused("too many", searches=65535, beams=32, vocab=1 << 20)
    refused("eos", eos=-2)
    refused("eos", eos=50000)
    for power in (-0.5, 17.0, float("nan"), float("inf")):
        refused("length_power", length_power=power)
    need = mmr.beam_select_workspace_size(2, 4, 50000)
    assert need > 0 and mmr.beam_select_workspace_size(2, 4, 100) == 0
    refused("too small", workspace=At(4096, need - 1))


def test_sizes_of_what_no_call_takes(mmr):
    """0 bytes, not the wrapped product."""
    assert mmr.kv8_fork_workspace_size(65535, 4096, 1 << 24) > 65535 * 4096 * 4
    for sizes in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (65536, 1, 1), (1, (1 << 24) + 1, 1), (1, 1, (1 << 24) + 1),
                  (65535, 1 << 14, 1), (1 << 62, 1 << 62, 5), (-1, 1, 1)):
        assert mmr.kv8_fork_workspace_size(*sizes) == 0, sizes
    for n in (0, -1, (1 << 24) + 1, 1 << 62):
        assert mmr.kv8_compact_workspace_size(n) == 0, n
    for sizes in ((0, 1, 1), (1, 33, 1), (1, 1, 1 << 62), (65535, 32, 1 << 24)):
        assert mmr.beam_select_workspace_size(*sizes) == 0, sizes


# ------------------------------------------------- the references themselves ----


def test_reference_fork_keeps_what_sequences_hold():
    """Whatever is forked: users count the table, every sequence reads its parent's tokens, and what it will write is
    its alone."""
    rng = np.random.default_rng(1)
    for _ in range(60):
        pool = paging.Pool(rng, 2, 40, 5, 6, 1, 4)
        tokens = rng.integers(0, 200, 5)
        pool.fill(rng, tokens, 0.4)
        for _ in range(4):
            parent = rng.integers(-1, 5, 5)
            keep = np.where(parent >= 0, np.minimum(tokens[parent], rng.integers(0, 250, 5)), 0)
            room = rng.integers(0, 90, 5)
            before, table = pool.keys.copy(), pool.table.copy()
            assert paging.fork(pool, parent, keep, room) in (0, paging.NO_PAGES)
            np.testing.assert_array_equal(pool.users, np.bincount(pool.table[pool.table >= 0], minlength=40))
            tokens = keep + room
            for s in range(5):
                places = -(-int(tokens[s]) // paging.PAGE)
                if (pool.table[s, :places] < 0).any():
                    tokens[s] = 0  # no more pages
                    continue
                for t in range(keep[s]):
                    was, now = table[parent[s], t // 64], pool.table[s, t // 64]
                    np.testing.assert_array_equal(pool.keys[:, now, :, t % 64], before[:, was, :, t % 64])
                if room[s]:
                    assert (pool.users[pool.table[s, keep[s] // 64: places]] == 1).all()


def test_reference_select_against_brute_force():
    rng = np.random.default_rng(2)
    for _ in range(50):
        beams, vocab = int(rng.integers(1, 5)), int(rng.integers(1, 9))
        logits = rng.integers(-2, 3, (beams, vocab)).astype(np.float32)
        scores = rng.integers(-3, 1, beams).astype(np.float32)
        ended, lengths = rng.integers(0, 2, beams), rng.integers(0, 5, beams)
        eos = int(rng.integers(-1, vocab))
        got, _, _ = paging.select(logits, beams, eos, 0.7, scores, lengths, ended)
        every = []
        for b in range(beams):
            p = np.exp(logits[b].astype(np.float64))
            for v in range(vocab):
                if eos >= 0 and ended[b]:
                    if v == eos:
                        every.append((float(scores[b]), max(int(lengths[b]), 1), b, v, 0.0))
                else:
                    every.append((scores[b] + np.log(p[v] / p.sum()), int(lengths[b]) + 1, b, v, float(logits[b, v])))
        every.sort(key=lambda c: (-round(c[0] * c[1] ** -0.7, 9), c[2], -c[4], c[3]))
        n = min(beams, len(every))
        assert list(zip(got[3][:n], got[4][:n])) == [(c[2], c[3]) for c in every[:n]]
        assert (got[3][n:] == -1).all()


def test_reference_window_of_everything(mmr):
    rng = np.random.default_rng(3)
    cache = ref.Cache(rng, 6, 2, 3, 2, 32)
    cache.fill(rng, [130, 70])
    query = rng.standard_normal((4, 4 * 32)).astype(np.float32)
    args = cache, query, [0, 1, 4], [129, 67], 4
    want, _ = ref.attention(*args, query)
    for sinks, window in ((0, 130), (130, 1), (100, 30)):
        got, _ = paging.window_attention(*args, sinks, window, query)
        np.testing.assert_allclose(got, want, atol=1e-12)
