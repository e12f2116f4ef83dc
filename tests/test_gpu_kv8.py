"""The 8-bit paged cache on the GPU against its definition in 64 bits: codes and
exponents bit for bit, queries to half a step, attention within the bound that
low_bit_reference.attention derives for each row."""
from __future__ import annotations

import numpy as np
import pytest

import low_bit_reference as ref

pytestmark = pytest.mark.gpu
THETA, EPS = 1e6, 1e-5
HALF_STEP = 2.0 ** -24


def ints(mmr, values):
    return mmr.DeviceArray.from_numpy(np.asarray(values, np.int32))


def pages_for(rows, context):
    return max(1, max(-(-(n + c) // ref.PAGE) for n, c in zip(rows, context)))


def offsets_of(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


class Append:
    """One append on the device and the same in 64 bits."""

    def __init__(self, mmr, cache, hq, norms=True, positions=32768, rng=None):
        self.mmr, self.cache, self.hq, d = mmr, cache, hq, cache.d
        self.rope = mmr.RopeTable(positions, d, THETA)
        self.norms = [(1 + 0.1 * rng.standard_normal(d)).astype(np.float32) if norms else None for _ in range(2)]
        self.dnorms = [mmr.DeviceArray.from_numpy(n) if norms else None for n in self.norms]
        self.device = cache.upload(mmr)
        self.error = ints(mmr, [0])

    def __call__(self, qkv, rows, context, stream=None, max_rows=None):
        mmr, offsets = self.mmr, offsets_of(rows)
        fill = np.full((len(qkv), self.hq * self.cache.d), 7.5, np.float32)
        query = mmr.DeviceArray.from_numpy(fill)
        mmr.kv8_append(mmr.DeviceArray.from_numpy(qkv), *self.dnorms, EPS, self.rope, self.device,
                       ints(mmr, offsets), ints(mmr, context), len(qkv), max_rows or max(rows), self.hq, query,
                       self.error, stream=stream)
        mmr.synchronize()
        want = ref.append(self.cache, qkv, offsets, context, self.hq, THETA, *self.norms, EPS, fill)
        return query.numpy(), want

    def check(self, qkv, rows, context, error=0):
        got, want = self(qkv, rows, context)
        self.cache.assert_equals(self.device)
        # Computed in 64 bits and rounded once.
        assert (np.abs(got - want) <= HALF_STEP * np.abs(want) + 1e-12).all()
        assert int(self.error.numpy()[0]) == error


def qkv_rows(rng, n, hq, hkv, d, std=0.6):
    return (rng.standard_normal((n, (hq + 2 * hkv) * d)) * std).astype(np.float32)


HEADS = [(8, 2, 96), (4, 4, 64), (8, 1, 128), (6, 2, 32)]


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("rows,context", [([1], [0]), ([1], [777]), ([1, 1, 1], [15, 16, 63]), ([5, 0, 17, 64], [3, 9, 60, 0]),
                                          ([130], [1]), ([16, 16], [16, 8])])
def test_append(gpu, hq, hkv, d, rows, context):
    print(f"[case] append {hq},{hkv},{d} rows {rows} context {context}", flush=True)
    rng = np.random.default_rng(sum(rows) * 31 + d)
    per = pages_for(rows, context)
    cache = ref.Cache(rng, len(rows) * per + 2, len(rows), per, hkv, d)
    cache.fill(rng, context)
    # Two rows behind the last sequence, whose queries stay as they are.
    Append(gpu, cache, hq, rng=rng).check(qkv_rows(rng, sum(rows) + 2, hq, hkv, d), rows, context)


@pytest.mark.parametrize("which", [0, 1])
def test_append_with_one_norm(gpu, which):
    rng = np.random.default_rng(51)
    cache = ref.Cache(rng, 4, 1, 4, 2, 96)
    step = Append(gpu, cache, 8, rng=rng)
    step.norms[which] = step.dnorms[which] = None
    step.check(qkv_rows(rng, 70, 8, 2, 96), [70], [3])


@pytest.mark.parametrize("hq,hkv,d", [(130, 1, 32), (64, 64, 32), (24, 3, 64)])
@pytest.mark.parametrize("rows,context", [([1, 1], [200, 30]), ([4, 70], [77, 0])])
def test_many_heads(gpu, hq, hkv, d, rows, context):
    """More heads than a tile of the attention has rows, and as many KV heads as there may be."""
    print(f"[case] heads {hq},{hkv},{d} rows {rows}", flush=True)
    rng = np.random.default_rng(hq + sum(rows))
    per = pages_for(rows, context)
    cache = ref.Cache(rng, 2 * per, 2, per, hkv, d)
    cache.fill(rng, context)
    Append(gpu, cache, hq, rng=rng).check(qkv_rows(rng, sum(rows), hq, hkv, d), rows, context)
    query = rng.standard_normal((sum(rows), hq * d)).astype(np.float32)
    check_attention(gpu, cache, query, rows, context, hq)


def test_rows_before_the_first_sequence(gpu):
    """offsets[0] above 0: the rows before it are nobody's, and stay."""
    mmr, rng = gpu, np.random.default_rng(53)
    hq, hkv, d = 8, 2, 96
    cache = ref.Cache(rng, 4, 2, 2, hkv, d)
    cache.fill(rng, [40, 3])
    step = Append(mmr, cache, hq, rng=rng)
    qkv, offsets, context = qkv_rows(rng, 20, hq, hkv, d), np.array([5, 6, 18], np.int32), [40, 3]
    fill = np.full((20, hq * d), 7.5, np.float32)
    query = mmr.DeviceArray.from_numpy(fill)
    mmr.kv8_append(mmr.DeviceArray.from_numpy(qkv), *step.dnorms, EPS, step.rope, step.device, ints(mmr, offsets),
                   ints(mmr, context), 20, 12, hq, query, step.error)
    want = ref.append(cache, qkv, offsets, context, hq, THETA, *step.norms, EPS, fill)
    cache.assert_equals(step.device)
    assert (np.abs(query.numpy() - want) <= HALF_STEP * np.abs(want) + 1e-12).all()
    q = query.numpy()
    got, error = attend(mmr, step.device, cache, q, offsets, context, hq, max_rows=12)
    want, bound = ref.attention(cache, q, offsets, context, hq, fill)
    assert error == 0 and int(step.error.numpy()[0]) == 0
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("seqs,rows", [(65535, 1), (9000, 3)])
def test_most_sequences_on_shared_pages(gpu, seqs, rows):
    """Every sequence has the same pages, one of them twice."""
    rng = np.random.default_rng(55)
    hq, hkv, d, kinds = 4, 2, 32, 5
    cache = ref.Cache(rng, kinds * 3, kinds, 3, hkv, d)
    cache.table[:] = [4, 9, 4]
    cache.fill(rng, [192] * kinds)
    context = np.array([0, 63, 64, 100, 188], np.int32)
    query = rng.standard_normal((kinds * rows, hq * d)).astype(np.float32)
    want, bound = ref.attention(cache, query, np.arange(kinds + 1) * rows, context, hq, query)
    kind = np.arange(seqs) % kinds
    row = (kind[:, None] * rows + np.arange(rows)).reshape(-1)
    good = cache.upload(gpu)
    table = gpu.DeviceArray.from_numpy(np.tile(cache.table[:1], (seqs, 1)))
    many = gpu.Kv8Pages(*good.buffers[:4], table, cache.pages, seqs, 3, hkv, d)
    cache.seqs = seqs
    got, error = attend(gpu, many, cache, query[row], np.arange(seqs + 1) * rows, context[kind], hq, max_rows=rows)
    assert error == 0
    assert (np.abs(got - want[row]) <= bound[row]).all()


def test_append_token_by_token_moves_blocks(gpu):
    """Every token larger than the ones before: the block's codes move to a larger exponent again and again."""
    rng = np.random.default_rng(5)
    cache = ref.Cache(rng, 3, 1, 2, 2, 96)
    step = Append(gpu, cache, 8, norms=False, rng=rng)
    for t in range(70):
        step.check(qkv_rows(rng, 1, 8, 2, 96, 1e-3 * 1.3 ** (t % 37)), [1], [t])


def test_append_sizes_at_both_ends(gpu):
    rng = np.random.default_rng(6)
    cache = ref.Cache(rng, 4, 1, 2, 2, 64)
    step = Append(gpu, cache, 4, norms=False, rng=rng)
    qkv = qkv_rows(rng, 80, 4, 2, 64)
    qkv[0:16] = 0.0
    qkv[16:32] *= 2.0 ** -130  # subnormal: the least exponent
    qkv[32:48] *= 2.0 ** 126
    qkv[48] = 127.0  # exactly on the border, and just past it
    qkv[49:64] = np.nextafter(np.float32(127.0), np.float32(200.0))
    qkv[64:80, ::3] = 0.5  # ties to even
    with np.errstate(over="ignore"):
        got, want = step(qkv, [80], [0])
    cache.assert_equals(step.device)
    assert int(step.error.numpy()[0]) == 0


def test_append_keeps_and_flags_what_is_not_finite(gpu):
    rng = np.random.default_rng(7)
    hq, hkv, d = 4, 2, 64
    cache = ref.Cache(rng, 4, 2, 2, hkv, d)
    step = Append(gpu, cache, hq, norms=False, rng=rng)
    qkv = qkv_rows(rng, 40, hq, hkv, d)
    v = (hq + hkv) * d
    qkv[3, v + 5], qkv[4, v + 6], qkv[5, v + d + 7] = np.inf, -np.inf, np.nan
    got, want = step(qkv, [20, 20], [0, 30])
    cache.assert_equals(step.device)
    assert int(step.error.numpy()[0]) == gpu.KV8_ERROR_NOT_FINITE
    assert np.isfinite(got).all()


def test_append_refuses_on_the_device(gpu):
    """Bad rows and pages are flagged; the other sequences are appended."""
    mmr, rng = gpu, np.random.default_rng(8)
    hq, hkv, d = 8, 2, 96
    cache = ref.Cache(rng, 12, 3, 3, hkv, d)
    cache.table[1, 1] = 12  # page past the pool
    step = Append(mmr, cache, hq, positions=150, rng=rng)
    before = [b.numpy() for b in step.device.buffers]
    qkv = qkv_rows(rng, 30, hq, hkv, d)
    offsets, context = [0, 10, 20, 30], [0, 64, 145]  # the last reaches past the rotation table
    query = mmr.DeviceArray.from_numpy(np.full((30, hq * d), 7.5, np.float32))
    mmr.kv8_append(mmr.DeviceArray.from_numpy(qkv), *step.dnorms, EPS, step.rope, step.device, ints(mmr, offsets),
                   ints(mmr, context), 30, 10, hq, query, step.error)
    assert int(step.error.numpy()[0]) == mmr.KV8_ERROR_ROWS
    got = query.numpy()
    assert (got[10:] == 7.5).all() and (got[:10] != 7.5).any(-1).all()
    for name, buffer, old in zip(("keys", "values", "key_exps", "value_exps"), step.device.buffers, before):
        now = buffer.numpy()
        now[cache.table[0, 0]] = old[cache.table[0, 0]]
        np.testing.assert_array_equal(now, old, err_msg=name)
    # Rows up to `fine` belong to a sequence that is in order.
    for offsets, rows, most, fine in (([0, 10, 5, 5], 30, 10, 10), ([0, 31, 31, 31], 30, 30, 0),
                                      ([0, 10, 10, 10], 30, 9, 0), ([-1, 0, 0, 0], 30, 9, 0)):
        step.error.zero()
        query.upload(np.full((30, hq * d), 7.5, np.float32))
        mmr.kv8_append(mmr.DeviceArray.from_numpy(qkv), *step.dnorms, EPS, step.rope, step.device,
                       ints(mmr, offsets), ints(mmr, [0, 0, 0]), rows, most, hq, query, step.error)
        assert int(step.error.numpy()[0]) == mmr.KV8_ERROR_ROWS, offsets
        got = query.numpy()
        assert (got[fine:] == 7.5).all() and (got[:fine] != 7.5).any(-1).all()


def test_append_at_far_positions(gpu):
    """Angles at positions near 2^24, on a table row of a quarter million pages that shares a few."""
    rng = np.random.default_rng(9)
    per, hq, hkv, d = 2 ** 18, 4, 2, 64
    cache = ref.Cache(rng, 5, 1, 1, hkv, d)
    cache.table = np.resize(cache.table, (1, per)).astype(np.int32)
    cache.table[0, -2:] = [3, 4]
    cache.per_seq = per
    context = [2 ** 24 - 70]
    Append(gpu, cache, hq, positions=2 ** 24, rng=rng).check(qkv_rows(rng, 70, hq, hkv, d), [70], context)


def attend(mmr, device, cache, query, offsets, context, hq, *, max_rows, max_tokens=None, stream=None, out=None):
    max_tokens = max_tokens or cache.per_seq * ref.PAGE
    size = mmr.kv8_attention_workspace_size(hq, cache.kv_heads, cache.d, cache.seqs, len(query), max_rows, max_tokens)
    out = out if out is not None else mmr.DeviceArray.from_numpy(np.full(query.shape, 7.5, np.float32))
    error = ints(mmr, [0])
    workspace = mmr.DeviceArray(size, np.uint8) if size else None
    mmr.kv8_attention(mmr.DeviceArray.from_numpy(query), device, ints(mmr, offsets), ints(mmr, context), len(query),
                      max_rows, max_tokens, hq, out, workspace, error, stream=stream)
    mmr.synchronize()
    return out.numpy(), int(error.numpy()[0])


def check_attention(mmr, cache, query, rows, context, hq):
    offsets = offsets_of(rows)
    got, error = attend(mmr, cache.upload(mmr), cache, query, offsets, context, hq, max_rows=max(rows))
    want, bound = ref.attention(cache, query, offsets, context, hq, np.full(query.shape, 7.5, np.float32))
    assert error == 0
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / np.maximum(bound, 1e-300)).max())
    inside = slice(0, int(offsets[-1]))
    # Rounding errors of either sign: sums over n pages are off by about sqrt(n), not n, half steps.
    norm = np.linalg.norm(got[inside] - want[inside]) / np.linalg.norm(want[inside])
    assert norm <= 4e-6, norm


@pytest.mark.parametrize("hq,hkv,d", HEADS + [(12, 4, 96), (16, 1, 64), (3, 3, 128)])
@pytest.mark.parametrize("rows,context", [
    ([1], [0]), ([1], [1]), ([1], [63]), ([1], [64]), ([1, 1, 1], [15, 777, 200]), ([1], [5000]),
    ([2, 1], [63, 700]), ([3, 0, 5], [100, 7, 511]), ([17, 2], [0, 130]), ([64], [0]), ([150], [77])])
def test_attention(gpu, hq, hkv, d, rows, context):
    print(f"[case] attention {hq},{hkv},{d} rows {rows} context {context}", flush=True)
    rng = np.random.default_rng(sum(rows) * 17 + sum(context) + d)
    per = pages_for(rows, context)
    cache = ref.Cache(rng, len(rows) * per + 1, len(rows), per, hkv, d)
    cache.fill(rng, [a + b for a, b in zip(rows, context)])
    query = rng.standard_normal((sum(rows) + 2, hq * d)).astype(np.float32)
    check_attention(gpu, cache, query, rows, context, hq)


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_attention_over_many_rows_of_blocks(gpu, rows):
    """Enough (sequence, tile) pairs that no split along the context is taken, and prompts of several waves a block."""
    rng = np.random.default_rng(rows)
    hq, hkv, d, seqs = 8, 8, 32, 130 if rows < 40 else 70
    context = [int(c) for c in rng.integers(0, 60 if rows == 40 else 200, seqs)]
    per = pages_for([rows] * seqs, context)
    cache = ref.Cache(rng, seqs * per, seqs, per, hkv, d)
    cache.fill(rng, [c + rows for c in context])
    check_attention(gpu, cache, rng.standard_normal((rows * seqs, hq * d)).astype(np.float32), [rows] * seqs, context,
                    hq)


@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 32), (4, 4, 64), (8, 2, 96), (6, 3, 128), (7, 1, 96)])
@pytest.mark.parametrize("rows,context", [([1, 1], [20000, 16300]), ([30], [9000])])
def test_attention_joins_many_splits(gpu, hq, hkv, d, rows, context):
    """As many splits as one join takes, and fewer of the second sequence; the same bits whenever it is called."""
    print(f"[case] joins {hq},{hkv},{d} rows {rows} context {context}", flush=True)
    rng = np.random.default_rng(sum(context) + d)
    per = pages_for(rows, context)
    cache = ref.Cache(rng, len(rows) * per, len(rows), per, hkv, d)
    cache.fill(rng, [a + b for a, b in zip(rows, context)])
    query = rng.standard_normal((sum(rows), hq * d)).astype(np.float32)
    check_attention(gpu, cache, query, rows, context, hq)
    device, offsets = cache.upload(gpu), offsets_of(rows)
    first, _ = attend(gpu, device, cache, query, offsets, context, hq, max_rows=max(rows))
    for _ in range(20):
        again, _ = attend(gpu, device, cache, query, offsets, context, hq, max_rows=max(rows))
        np.testing.assert_array_equal(again, first)


@pytest.mark.parametrize("rows", [1, 9])
def test_attention_over_values_of_any_size(gpu, rows):
    """Blocks whose values are 2^40 apart, all zero, or at the ends of the exponents; peaked and flat rows."""
    rng = np.random.default_rng(rows + 20)
    hq, hkv, d, n = 8, 2, 96, 700
    cache = ref.Cache(rng, 12, 1, 12, hkv, d)
    cache.fill(rng, [n + rows])
    cache.value_exps[cache.table[0, 2:4]] += 40
    cache.value_exps[cache.table[0, 5]] = -126
    cache.values[cache.table[0, 6]] = 0
    cache.key_exps[cache.table[0, 7]] -= 30
    query = rng.standard_normal((rows, hq * d)).astype(np.float32)
    query[:, :d] *= 30.0   # one key takes nearly all
    query[:, d:2 * d] = 0  # all keys alike
    query[:, 2 * d:3 * d] *= 1e-30
    check_attention(gpu, cache, query, [rows], [n], hq)
    # Without the large blocks the small ones must come out as exactly.
    cache.value_exps[:] = -60
    check_attention(gpu, cache, query, [rows], [n], hq)


@pytest.mark.parametrize("rows", [1, 20])
def test_attention_rows_that_are_not_finite(gpu, rows):
    rng = np.random.default_rng(31)
    hq, hkv, d = 8, 2, 64
    cache = ref.Cache(rng, 8, 2, 4, hkv, d)
    cache.fill(rng, [100 + rows, 130 + rows])
    query = rng.standard_normal((2 * rows, hq * d)).astype(np.float32)
    device, offsets = cache.upload(gpu), offsets_of([rows, rows])
    want, bound = ref.attention(cache, query, offsets, [100, 130], hq, query)
    bad = query.copy()
    bad[0, 3], bad[rows, d + 5], bad[-1, 5 * d] = np.nan, np.inf, -np.inf
    got, error = attend(gpu, device, cache, bad, offsets, [100, 130], hq, max_rows=rows)
    assert error == 0
    mask = np.zeros(want.shape, bool)
    mask[0, :d] = mask[rows, d:2 * d] = mask[-1, 5 * d:6 * d] = True
    assert np.isnan(got[mask]).all()
    assert (np.abs(got - want) <= bound)[~mask].all()


def test_attention_takes_keys_of_bad_pages_as_absent(gpu):
    rng = np.random.default_rng(33)
    hq, hkv, d = 8, 2, 96
    cache = ref.Cache(rng, 12, 2, 4, hkv, d)
    cache.fill(rng, [200, 64])
    query = rng.standard_normal((2, hq * d)).astype(np.float32)
    good = cache.upload(gpu)
    table = cache.table.copy()
    table[0, 1], table[1, 0] = -1, 12  # of the second sequence nothing is left: a row of zeros
    bad = gpu.Kv8Pages(*good.buffers[:4], ints(gpu, table), 12, 2, 4, hkv, d)
    got, error = attend(gpu, bad, cache, query, [0, 1, 2], [199, 63], hq, max_rows=1)
    assert error == gpu.KV8_ERROR_ROWS and (got[1] == 0).all()
    short = ref.Cache(rng, 12, 1, 4, hkv, d)  # the same keys without that page
    short.keys, short.values, short.key_exps, short.value_exps = (
        cache.keys, cache.values, cache.key_exps, cache.value_exps)
    short.table = cache.table[:1, [0, 2, 3, 1]].copy()
    want, bound = ref.attention(short, query[:1], [0, 1], [199 - 64], hq, query[:1])
    assert (np.abs(got[0] - want[0]) <= bound[0]).all()
    # More keys than the launch was sized for, and offsets that fall: nothing is written.
    for offsets, context, tokens in (([0, 1, 2], [199, 63], 150), ([1, 0, 2], [199, 63], 256)):
        got, error = attend(gpu, good, cache, query, offsets, context, hq, max_rows=1, max_tokens=tokens)
        assert error == gpu.KV8_ERROR_ROWS and (got[0] == 7.5).all()


def test_pages_past_four_gigabytes(gpu):
    mmr, rng = gpu, np.random.default_rng(35)
    hq, hkv, d, pages = 8, 2, 128, 300_000  # 4.9 GB of codes each
    small = ref.Cache(rng, 3, 1, 3, hkv, d)
    at = np.array([[pages - 1, 7, pages - 9]], np.int32)
    big = mmr.Kv8Pages(mmr.DeviceArray((pages, hkv, 64, d), np.int8), mmr.DeviceArray((pages, hkv, d, 64), np.int8),
                       mmr.DeviceArray((pages, hkv, 4), np.int8), mmr.DeviceArray((pages, hkv, 4), np.int8),
                       ints(mmr, at), pages, 1, 3, hkv, d)
    step = Append(mmr, small, hq, rng=rng)
    twin = step.device
    step.device = big
    query, want = step(qkv_rows(rng, 140, hq, hkv, d), [140], [0])
    assert (np.abs(query - want) <= HALF_STEP * np.abs(want) + 1e-12).all()
    got, error = attend(mmr, big, small, query, [0, 140], [0], hq, max_rows=140)
    want, bound = ref.attention(small, query, [0, 140], [0], hq, query)
    assert error == 0 and (np.abs(got - want) <= bound).all()
    del twin


def test_recorded_steps_follow_the_device_arrays(gpu):
    """Append and attention in one graph, replayed with contexts and pages advanced in device memory, against the same
    calls made eagerly on another stream; two graphs with workspaces of their own, replayed in turn."""
    mmr, rng = gpu, np.random.default_rng(37)
    hq, hkv, d, seqs, per = 8, 2, 96, 3, 8
    twins = []
    for stream in (mmr.Stream(), mmr.Stream(), mmr.Stream()):
        r = np.random.default_rng(39)
        cache = ref.Cache(r, seqs * per, seqs, per, hkv, d)
        cache.fill(r, [40, 15, 300])
        step = Append(mmr, cache, hq, rng=r)
        size = mmr.kv8_attention_workspace_size(hq, hkv, d, seqs, seqs, 1, per * 64)
        t = dict(step=step, stream=stream, qkv=mmr.DeviceArray((seqs, (hq + 2 * hkv) * d), np.float32),
                 offsets=ints(mmr, [0, 1, 2, 3]), context=ints(mmr, [0, 0, 0]),
                 query=mmr.DeviceArray((seqs, hq * d), np.float32), out=mmr.DeviceArray((seqs, hq * d), np.float32),
                 workspace=mmr.DeviceArray(max(size, 1), np.uint8))
        twins.append(t)

    def calls(t):
        s = t["step"]
        mmr.kv8_append(t["qkv"], *s.dnorms, EPS, s.rope, s.device, t["offsets"], t["context"], seqs, 1, hq, t["query"],
                       s.error, stream=t["stream"])
        mmr.kv8_attention(t["query"], s.device, t["offsets"], t["context"], seqs, 1, per * 64, hq, t["out"],
                          t["workspace"], s.error, stream=t["stream"])

    graphs = []
    for t in twins[:2]:
        with mmr.Graph(t["stream"]) as g:
            calls(t)
        graphs.append(g)
    for step in range(20):
        qkv = qkv_rows(rng, seqs, hq, hkv, d)
        for t in twins:
            t["qkv"].upload(qkv)
            t["context"].upload(np.array([40 + step, 15 + step, 300 + step], np.int32))
        calls(twins[2])
        for t, g in zip(twins, graphs):
            g.launch(t["stream"])
        mmr.synchronize()
        for t in twins[:2]:
            for name in ("query", "out"):
                np.testing.assert_array_equal(t[name].numpy(), twins[2][name].numpy(), err_msg=f"{name} step {step}")
            for a, b in zip(t["step"].device.buffers, twins[2]["step"].device.buffers):
                np.testing.assert_array_equal(a.numpy(), b.numpy())


def test_no_rows_is_no_work(gpu):
    mmr, rng = gpu, np.random.default_rng(41)
    cache = ref.Cache(rng, 2, 1, 2, 2, 96)
    step = Append(mmr, cache, 8, rng=rng)
    one = mmr.DeviceArray.from_numpy(np.full((1, 1152), 7.5, np.float32))
    for rows in (0, 1):
        mmr.kv8_append(one, *step.dnorms, EPS, step.rope, step.device, ints(mmr, [0, 0]), ints(mmr, [128]), rows, 0, 8,
                       one, step.error)
        mmr.kv8_attention(one, step.device, ints(mmr, [0, 0]), ints(mmr, [128]), rows, 0, 128, 8, one, None,
                          step.error)
    # A sequence without rows in a launch that could have brought one; its context may be the whole table.
    mmr.kv8_append(one, *step.dnorms, EPS, step.rope, step.device, ints(mmr, [0, 0]), ints(mmr, [128]), 1, 1, 8, one,
                   step.error)
    got, error = attend(mmr, step.device, cache, np.zeros((1, 768), np.float32), [0, 0], [128], 8, max_rows=1)
    mmr.synchronize()
    assert error == 0 and (got == 7.5).all() and (one.numpy() == 7.5).all() and int(step.error.numpy()[0]) == 0
    cache.assert_equals(step.device)


def test_thousands_of_sequences(gpu):
    """One row each, on caches of one to three pages, in one call."""
    rng = np.random.default_rng(43)
    seqs, per, hq, hkv, d = 3000, 3, 2, 1, 32
    cache = ref.Cache(rng, seqs * per, seqs, per, hkv, d)
    context = [int(c) for c in rng.integers(0, 190, seqs)]
    step = Append(gpu, cache, hq, rng=rng)
    step.check(qkv_rows(rng, seqs, hq, hkv, d), [1] * seqs, context)
    # Cached tokens before the new rows are whatever the pages held: their exponents can be anything a block may have.
    cache.key_exps[:] = np.clip(cache.key_exps, -12, -4)
    cache.value_exps[:] = np.clip(cache.value_exps, -12, -4)
    check_attention(gpu, cache, rng.standard_normal((seqs, hq * d)).astype(np.float32), [1] * seqs, context, hq)


def test_calls_on_two_streams_at_once(gpu):
    """Caches, workspaces and errors of their own: neither call sees the other."""
    mmr = gpu
    runs = []
    for seed in (45, 46):
        rng = np.random.default_rng(seed)
        cache = ref.Cache(rng, 2 * 20, 2, 20, 2, 96)
        cache.fill(rng, [1200, 700])
        query = rng.standard_normal((2, 8 * 96)).astype(np.float32)
        size = mmr.kv8_attention_workspace_size(8, 2, 96, 2, 2, 1, 1280)
        runs.append(dict(cache=cache, device=cache.upload(mmr), query=query, dq=mmr.DeviceArray.from_numpy(query),
                         out=mmr.DeviceArray((2, 768), np.float32), ws=mmr.DeviceArray(size, np.uint8),
                         offsets=ints(mmr, [0, 1, 2]), context=ints(mmr, [1199, 699]), error=ints(mmr, [0]),
                         stream=mmr.Stream()))
    mmr.synchronize()
    for _ in range(20):
        for r in runs:
            mmr.kv8_attention(r["dq"], r["device"], r["offsets"], r["context"], 2, 1, 1280, 8, r["out"], r["ws"],
                              r["error"], stream=r["stream"])
    mmr.synchronize()
    for r in runs:
        want, bound = ref.attention(r["cache"], r["query"], [0, 1, 2], [1199, 699], 8, r["query"])
        assert (np.abs(r["out"].numpy() - want) <= bound).all()


@pytest.mark.parametrize("rows,context", [([1, 1], [100, 2000]), ([2, 2], [100, 2000]), ([40, 90], [3, 600])])
def test_out_in_place_of_the_query(gpu, rows, context):
    mmr, rng = gpu, np.random.default_rng(47)
    per = pages_for(rows, context)
    cache = ref.Cache(rng, 2 * per, 2, per, 2, 64)
    cache.fill(rng, [a + b for a, b in zip(rows, context)])
    query = rng.standard_normal((sum(rows), 8 * 64)).astype(np.float32)
    both, error, max_rows = mmr.DeviceArray.from_numpy(query), ints(mmr, [0]), max(rows)
    size = mmr.kv8_attention_workspace_size(8, 2, 64, 2, len(query), max_rows, per * 64)
    mmr.kv8_attention(both, cache.upload(mmr), ints(mmr, offsets_of(rows)), ints(mmr, context), len(query), max_rows,
                      per * 64, 8, both, mmr.DeviceArray(max(size, 1), np.uint8), error)
    want, bound = ref.attention(cache, query, offsets_of(rows), context, 8, query)
    assert (np.abs(both.numpy() - want) <= bound).all()


# (query heads, KV heads), rows and context: steps of one and of two blocks, and the kernel for many rows.
BORDERS = [(2, 2, 2, 15), (2, 2, 4, 30), (2, 2, 3, 62), (4, 2, 3, 47), (2, 1, 4, 126), (4, 1, 9, 60), (6, 2, 20, 700),
           (1, 1, 40, 8)]


@pytest.mark.parametrize("hq,hkv,rows,context", BORDERS)
@pytest.mark.parametrize("larger", [20, 28, 40])
def test_attention_rows_before_far_larger_values(gpu, hq, hkv, rows, context, larger):
    """A later row opens a block whose values are far larger: the rows that do not attend it lose nothing."""
    print(f"[case] borders {hq},{hkv} rows {rows} context {context} larger {larger}", flush=True)
    rng = np.random.default_rng(rows * 7 + context + larger)
    per = pages_for([rows], [context])
    cache = ref.Cache(rng, per, 1, per, hkv, 64)
    cache.fill(rng, [rows + context])
    for block in range(context // ref.BLOCK + 1, (context + rows - 1) // ref.BLOCK + 1):
        # Each block that the rows open, larger than the one before.
        cache.value_exps[cache.table[0, block * ref.BLOCK // ref.PAGE], :, block % 4] = (
            -6 + larger * (block - context // ref.BLOCK))
    query = rng.standard_normal((rows, hq * 64)).astype(np.float32)
    got, error = attend(gpu, cache.upload(gpu), cache, query, [0, rows], [context], hq, max_rows=rows)
    want, bound = ref.attention(cache, query, [0, rows], [context], hq, query)
    assert error == 0
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / np.maximum(bound, 1e-300)).max())


@pytest.mark.parametrize("rows,context", [(2, 300), (2, 1000), (10, 300), (23, 1500)])
def test_attention_rows_do_not_depend_on_rows_of_other_blocks(gpu, rows, context):
    """Three heads a KV head: a group's last rows share a block of four or a wave of 16 with places that no row has,
    and their bits are the same whatever the rows of other blocks ask for."""
    rng = np.random.default_rng(rows)
    hkv, d, per = 4, 64, pages_for([rows], [context])
    cache = ref.Cache(rng, per, 1, per, hkv, d)
    cache.fill(rng, [rows + context])
    device = cache.upload(gpu)
    query = rng.standard_normal((rows, 3 * hkv * d)).astype(np.float32)
    other = query.copy()
    other[0] = 60.0 * rng.standard_normal(3 * hkv * d)
    both = [attend(gpu, device, cache, q, [0, rows], [context], 3 * hkv, max_rows=rows)[0] for q in (query, other)]
    # [KV head][row (token, head) of the group][d]
    both = [o.reshape(rows, hkv, 3, d).swapaxes(0, 1).reshape(hkv, rows * 3, d) for o in both]
    part = 4 if rows * 3 <= 8 else 16
    assert rows * 3 % part, "places without a row"
    last = rows * 3 // part * part
    np.testing.assert_array_equal(both[0][:, last:], both[1][:, last:])


@pytest.mark.parametrize("rows", [1, 3, 20])
@pytest.mark.parametrize("power", [60, 100, 120])
def test_attention_of_tiny_queries_and_large_keys(gpu, rows, power):
    """Scores of ordinary size, whatever the sizes of what they are products of; and the other way round."""
    rng = np.random.default_rng(rows + power)
    hq, hkv, d, n = 4, 2, 64, 300
    for sign in (1, -1):
        cache = ref.Cache(rng, 6, 1, 6, hkv, d)
        cache.fill(rng, [n + rows])
        cache.key_exps = np.clip(cache.key_exps + np.int64(sign * power), -126, 122).astype(np.int8)
        query = np.ldexp(rng.standard_normal((rows, hq * d)), -sign * power).astype(np.float32)
        check_attention(gpu, cache, query, [rows], [n], hq)


def test_prompts_and_steps_in_two_calls_on_the_same_arrays(gpu):
    """Sequences with prompts first: a call for them, and one from the first of the others on, each with max_rows of its
    own; neither touches the other's rows."""
    mmr, rng = gpu, np.random.default_rng(57)

    class From:
        def __init__(self, array, elements):
            self.ptr, self.nbytes = array.ptr + 4 * elements, array.nbytes - 4 * elements

    hq, hkv, d, rows, context = 8, 2, 96, [70, 33, 1, 1, 2, 1], [5, 0, 400, 15, 700, 64]
    per, prompts, total = pages_for(rows, context), 2, sum(rows)
    cache = ref.Cache(rng, 6 * per, 6, per, hkv, d)
    cache.fill(rng, [a + b for a, b in zip(rows, context)])
    query = rng.standard_normal((total, hq * d)).astype(np.float32)
    fill = np.full(query.shape, 7.5, np.float32)
    device, out, error = cache.upload(mmr), mmr.DeviceArray.from_numpy(fill), ints(mmr, [0])
    dq, offsets, dcontext = mmr.DeviceArray.from_numpy(query), ints(mmr, offsets_of(rows)), ints(mmr, context)
    want, bound = ref.attention(cache, query, offsets_of(rows), context, hq, fill)
    for first, seqs, max_rows in ((0, prompts, 70), (prompts, 6 - prompts, 2)):
        pages = mmr.Kv8Pages(*device.buffers[:4], From(device.buffers[4], first * per), cache.pages, seqs, per, hkv, d)
        size = mmr.kv8_attention_workspace_size(hq, hkv, d, seqs, total, max_rows, per * ref.PAGE)
        mmr.kv8_attention(dq, pages, From(offsets, first), From(dcontext, first), total, max_rows, per * ref.PAGE, hq, out,
                          mmr.DeviceArray(max(size, 1), np.uint8), error)
        got, done = out.numpy(), sum(rows[: first + seqs])
        assert (np.abs(got - want) <= bound)[:done].all() and (got[done:] == 7.5).all()
    assert int(error.numpy()[0]) == 0
