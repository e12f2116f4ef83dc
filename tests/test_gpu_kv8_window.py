"""Attention with a window and sinks over the 8-bit cache against 64 bits, within the bound that
low_bit_reference.attention derives, over the keys that each row attends."""
from __future__ import annotations

import numpy as np
import pytest

import low_bit_reference as ref
import paging_reference as paging
from test_gpu_kv8 import HEADS, ints, offsets_of, pages_for

pytestmark = pytest.mark.gpu


def attend(mmr, device, cache, query, offsets, context, hq, sinks, window, *, max_rows, max_tokens=None, out=None,
           stream=None):
    max_tokens = max_tokens or cache.per_seq * ref.PAGE
    size = mmr.kv8_window_attention_workspace_size(hq, cache.kv_heads, cache.d, cache.seqs, len(query), max_rows,
                                                   max_tokens, sinks, window)
    out = out if out is not None else mmr.DeviceArray.from_numpy(np.full(query.shape, 7.5, np.float32))
    error = ints(mmr, [0])
    workspace = mmr.DeviceArray(size, np.uint8) if size else None
    mmr.kv8_window_attention(mmr.DeviceArray.from_numpy(query), device, ints(mmr, offsets), ints(mmr, context),
                             len(query), max_rows, max_tokens, sinks, window, hq, out, workspace, error,
                             stream=stream)
    mmr.synchronize()
    return out.numpy(), int(error.numpy()[0])


def check(mmr, cache, query, rows, context, hq, sinks, window, device=None):
    offsets = offsets_of(rows)
    got, error = attend(mmr, device or cache.upload(mmr), cache, query, offsets, context, hq, sinks, window,
                        max_rows=max(rows))
    want, bound = paging.window_attention(cache, query, offsets, context, hq, sinks, window,
                                          np.full(query.shape, 7.5, np.float32))
    assert error == 0
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / np.maximum(bound, 1e-300)).max())
    return got


def without_unseen_pages(mmr, cache, rows, context, sinks, window):
    """The cache on the device with no numbers for the pages that no row attends."""
    table = cache.table.copy()
    for s in range(cache.seqs):
        for p in range(cache.per_seq):
            last = p * ref.PAGE + ref.PAGE - 1
            if last < context[s] - window + 1 and p * ref.PAGE >= sinks or p * ref.PAGE >= context[s] + rows[s]:
                table[s, p] = -1 if p % 2 else cache.pages + 5
    return mmr.Kv8Pages(*cache.upload(mmr).buffers[:4], ints(mmr, table), cache.pages, cache.seqs, cache.per_seq,
                        cache.kv_heads, cache.d)


CASES = [
    ([1], [0], 0, 1), ([1], [63], 1, 1), ([1], [64], 4, 64), ([1], [200], 0, 1), ([1, 1, 1], [15, 777, 200], 4, 100),
    ([1], [5000], 4, 1000), ([1], [5000], 130, 64), ([1], [5000], 63, 4900), ([1, 1], [4999, 70], 0, 3000),
    ([2, 1], [63, 700], 65, 129), ([2], [1023], 0, 3), ([3, 0, 5], [100, 7, 511], 16, 50), ([8], [130], 0, 65),
    ([17, 2], [0, 130], 4, 7), ([64], [0], 0, 1), ([64], [3], 1, 16), ([150], [77], 20, 100), ([150], [900], 64, 64),
    ([200], [4000], 4, 1500), ([33, 200], [1000, 0], 100, 90),
]


@pytest.mark.parametrize("hq,hkv,d", HEADS + [(12, 4, 96), (16, 1, 64), (3, 3, 128)])
@pytest.mark.parametrize("rows,context,sinks,window", CASES)
def test_window(gpu, hq, hkv, d, rows, context, sinks, window):
    print(f"[case] window {hq},{hkv},{d} rows {rows} context {context} sinks {sinks} window {window}", flush=True)
    rng = np.random.default_rng(sum(rows) * 17 + sum(context) + d)
    per = pages_for(rows, context) + 1
    cache = ref.Cache(rng, len(rows) * per + 1, len(rows), per, hkv, d)
    cache.fill(rng, [a + b for a, b in zip(rows, context)])
    query = rng.standard_normal((sum(rows) + 2, hq * d)).astype(np.float32)
    device = without_unseen_pages(gpu, cache, rows, context, sinks, window)
    check(gpu, cache, query, rows, context, hq, sinks, window, device)


@pytest.mark.parametrize("seed", range(12))
def test_windows_of_any_size(gpu, seed):
    rng = np.random.default_rng(100 + seed)
    hq, hkv, d = [(8, 2, 96), (8, 2, 64), (4, 4, 32), (8, 1, 128)][seed % 4]
    seqs, most = int(rng.integers(1, 5)), int(rng.choice([1, 2, 5, 40, 130]))
    rows = [int(n) for n in rng.integers(0, most + 1, seqs)]
    rows[0] = most
    context = [int(n) for n in rng.integers(0, 1500, seqs)]
    per = pages_for(rows, context) + 1
    cache = ref.Cache(rng, seqs * per, seqs, per, hkv, d)
    cache.fill(rng, [a + b for a, b in zip(rows, context)])
    query = rng.standard_normal((sum(rows), hq * d)).astype(np.float32)
    for _ in range(4):
        sinks, window = int(rng.integers(0, 200)), int(np.exp(rng.uniform(0, 7.4)))
        print(f"[case] {rows} {context} {hq},{hkv},{d} sinks {sinks} window {window}", flush=True)
        device = without_unseen_pages(gpu, cache, rows, context, sinks, window)
        check(gpu, cache, query, rows, context, hq, sinks, window, device)


@pytest.mark.parametrize("rows,context", [([1, 1], [700, 64]), ([5], [3000]), ([70], [400])])
def test_window_of_everything_is_attention(gpu, rows, context):
    """The same bits as the call without a window."""
    rng = np.random.default_rng(sum(context))
    hq, hkv, d, per = 8, 2, 96, pages_for(rows, context)
    cache = ref.Cache(rng, len(rows) * per, len(rows), per, hkv, d)
    cache.fill(rng, [a + b for a, b in zip(rows, context)])
    query, offsets = rng.standard_normal((sum(rows), hq * d)).astype(np.float32), offsets_of(rows)
    from test_gpu_kv8 import attend as whole

    device = cache.upload(gpu)
    want, _ = whole(gpu, device, cache, query, offsets, context, hq, max_rows=max(rows))
    for sinks, window in ((0, per * 64), (5, 1 << 40), (per * 64, 1), (1 << 50, 3)):
        got, error = attend(gpu, device, cache, query, offsets, context, hq, sinks, window, max_rows=max(rows))
        assert error == 0
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("rows", [1, 20])
def test_window_hides_values_of_any_size(gpu, rows):
    """What a row does not attend does not touch its sums: neither keys and values far larger than its own, nor blocks
    under any exponent, in pages that it attends other keys of."""
    rng = np.random.default_rng(rows)
    hq, hkv, d, context, sinks, window = 8, 2, 96, 800, 20, 150
    cache = ref.Cache(rng, 20, 1, 20, hkv, d)
    cache.fill(rng, [context + rows])
    query = rng.standard_normal((rows, hq * d)).astype(np.float32)
    first = context - window + 1
    # Blocks between the sinks and the window of the first row.
    for block in range(-(-sinks // 16), first // 16):
        page = cache.table[0, block // 4]
        cache.key_exps[page, :, block % 4] = cache.value_exps[page, :, block % 4] = 122 if block % 2 else -128
        cache.keys[page, :, block % 4 * 16: block % 4 * 16 + 16] = 127
    check(gpu, cache, query, [rows], [context], hq, sinks, window)
    # Of the sinks' own block, the tokens that are none.
    page = cache.table[0, 0]
    cache.keys[page, :, sinks:32], cache.values[page, :, :, sinks:32] = -128, 127
    check(gpu, cache, query, [rows], [context], hq, sinks, window)


@pytest.mark.parametrize("rows", [1, 20])
def test_window_rows_that_are_not_finite(gpu, rows):
    rng = np.random.default_rng(31)
    hq, hkv, d = 8, 2, 64
    cache = ref.Cache(rng, 16, 2, 8, hkv, d)
    cache.fill(rng, [400 + rows, 330 + rows])
    query, offsets = rng.standard_normal((2 * rows, hq * d)).astype(np.float32), offsets_of([rows, rows])
    want, bound = paging.window_attention(cache, query, offsets, [400, 330], hq, 4, 90, query)
    query[0, 3], query[rows, d + 5], query[-1, 5 * d] = np.nan, np.inf, -np.inf
    got, error = attend(gpu, cache.upload(gpu), cache, query, offsets, [400, 330], hq, 4, 90, max_rows=rows)
    mask = np.zeros(want.shape, bool)
    mask[0, :d] = mask[rows, d:2 * d] = mask[-1, 5 * d:6 * d] = True
    assert error == 0 and np.isnan(got[mask]).all()
    assert (np.abs(got - want) <= bound)[~mask].all()


def test_window_takes_keys_of_bad_pages_as_absent(gpu):
    """A page that rows attend without a number is flagged; where a row has no key left, it is zeros."""
    rng = np.random.default_rng(33)
    hq, hkv, d = 8, 2, 96
    cache = ref.Cache(rng, 24, 2, 12, hkv, d)
    cache.fill(rng, [700, 640])
    query = rng.standard_normal((2, hq * d)).astype(np.float32)
    good = cache.upload(gpu)
    table = cache.table.copy()
    table[0, 10], table[1, 9] = -1, 24  # of the second sequence's window nothing is left
    bad = gpu.Kv8Pages(*good.buffers[:4], ints(gpu, table), 24, 2, 12, hkv, d)
    got, error = attend(gpu, bad, cache, query, [0, 1, 2], [703, 639], hq, 0, 64, max_rows=1)
    assert error == gpu.KV8_ERROR_ROWS and (got[1] == 0).all() and (got[0] == 0).all()
    # The first sequence has 36 keys of page 9 and 64 of page 10: those of page 9 are left.
    got, error = attend(gpu, bad, cache, query, [0, 1, 2], [703, 639], hq, 0, 100, max_rows=1)
    assert error == gpu.KV8_ERROR_ROWS
    short = ref.Cache(rng, 24, 1, 12, hkv, d)
    short.keys, short.values, short.key_exps, short.value_exps = (cache.keys, cache.values, cache.key_exps,
                                                                  cache.value_exps)
    short.table = cache.table[:1].copy()
    want, bound = paging.window_attention(short, query[:1], [0, 1], [639], hq, 0, 36, query[:1])
    assert (np.abs(got[0] - want[0]) <= bound[0]).all()
    for offsets, context, tokens in (([0, 1, 2], [703, 639], 650), ([1, 0, 2], [703, 639], 768)):
        got, error = attend(gpu, good, cache, query, offsets, context, hq, 4, 100, max_rows=1, max_tokens=tokens)
        assert error == gpu.KV8_ERROR_ROWS and (got[0] == 7.5).all()


def test_window_at_far_positions(gpu):
    """The end of a context of 2^24 tokens, on a table row of a quarter million pages of which a few have numbers."""
    rng = np.random.default_rng(35)
    per, hq, hkv, d = 2 ** 18, 8, 2, 64
    cache = ref.Cache(rng, 12, 1, 12, hkv, d)
    cache.fill(rng, [768])
    near = cache.table[0].copy()
    cache.table = np.full((1, per), -1, np.int32)
    cache.table[0, :2], cache.table[0, -10:] = near[:2], near[2:]
    cache.per_seq = per
    device = cache.upload(gpu)
    for rows, sinks, window in ((1, 100, 500), (5, 128, 600), (40, 0, 550)):
        context = per * 64 - rows
        query = rng.standard_normal((rows, hq * d)).astype(np.float32)
        got, error = attend(gpu, device, cache, query, [0, rows], [context], hq, sinks, window, max_rows=rows)
        # The same keys, close together: moved by whole pages, so that sinks, window and causality hold as they did.
        short = ref.Cache(rng, 12, 1, 12, hkv, d)
        short.keys, short.values, short.key_exps, short.value_exps = (cache.keys, cache.values, cache.key_exps,
                                                                      cache.value_exps)
        short.table = near[None]
        want, bound = paging.window_attention(short, query, [0, rows], [768 - rows], hq, sinks, window, query)
        assert error == 0 and (np.abs(got - want) <= bound).all()


def test_window_in_place_and_always_the_same(gpu):
    mmr, rng = gpu, np.random.default_rng(37)
    hq, hkv, d = 8, 2, 96
    for rows, context, window in ([1, 1], [9000, 5000], 8000), ([90], [500], 200), ([5, 3], [6000, 100], 5000):
        per = pages_for(rows, context)
        cache = ref.Cache(rng, len(rows) * per, len(rows), per, hkv, d)
        cache.fill(rng, [a + b for a, b in zip(rows, context)])
        query, device = rng.standard_normal((sum(rows), hq * d)).astype(np.float32), cache.upload(mmr)
        first = check(mmr, cache, query, rows, context, hq, 4, window, device)
        size = mmr.kv8_window_attention_workspace_size(hq, hkv, d, len(rows), sum(rows), max(rows), per * 64, 4, window)
        workspace = mmr.DeviceArray(max(size, 1), np.uint8)
        args = ints(mmr, offsets_of(rows)), ints(mmr, context)
        error, both = ints(mmr, [0]), mmr.DeviceArray.from_numpy(query)
        for _ in range(10):
            both.upload(query)
            mmr.kv8_window_attention(both, device, *args, sum(rows), max(rows), per * 64, 4, window, hq, both, workspace,
                                     error)
            mmr.synchronize()
            np.testing.assert_array_equal(both.numpy(), first)


def test_recorded_windows_share_a_workspace(gpu):
    """Recorded calls of several forms on one workspace, replayed in changing order with eager calls between."""
    mmr, rng, stream = gpu, np.random.default_rng(39), gpu.Stream()
    hq, hkv, d, per = 8, 2, 96, 60
    cache = ref.Cache(rng, 3 * per, 3, per, hkv, d)
    cache.fill(rng, [3800, 700, 130])
    device, calls = cache.upload(mmr), []
    for rows, context, sinks, window in (([1, 1, 1], [3799, 699, 129], 4, 3000), ([30, 40, 20], [3770, 660, 110], 70, 600),
                                         ([1, 0, 5], [3799, 5, 100], 0, 2900)):
        n, offsets = sum(rows), offsets_of(rows)
        query = rng.standard_normal((n, hq * d)).astype(np.float32)
        args = [mmr.DeviceArray.from_numpy(query), device, ints(mmr, offsets), ints(mmr, context), n, max(rows), per * 64,
                sinks, window, hq, mmr.DeviceArray((n, hq * d), np.float32)]
        size = mmr.kv8_window_attention_workspace_size(hq, hkv, d, 3, n, max(rows), per * 64, sinks, window)
        calls.append((args, size, check(mmr, cache, query, rows, context, hq, sinks, window, device)))
    workspace, error, graphs = mmr.DeviceArray(max(c[1] for c in calls), np.uint8), ints(mmr, [0]), []
    assert min(c[1] for c in calls) > 0
    for args, _, _ in calls:
        with mmr.Graph(stream) as graph:
            mmr.kv8_window_attention(*args, workspace, error, stream=stream)
        graphs.append(graph)
    for order in ([0, 1, 2], [2, 1, 0], [1, 1, 0, 2], [0, 2, 0, 1]):
        for args, _, _ in calls:
            args[-1].zero()
        workspace.upload(np.full(workspace.shape, 0xFF, np.uint8))
        mmr.synchronize()
        for i in order:
            graphs[i].launch(stream)
        mmr.kv8_window_attention(*calls[order[0]][0], workspace, error, stream=stream)
        mmr.synchronize()
        for args, _, want in calls:
            np.testing.assert_array_equal(args[-1].numpy(), want)
    assert int(error.numpy()[0]) == 0
