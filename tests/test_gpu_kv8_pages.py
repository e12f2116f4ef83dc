"""Forking and compacting the pages of the 8-bit cache: tables, users and every byte of every page as the definition
has them."""
from __future__ import annotations

import numpy as np
import pytest

import paging_reference as paging

pytestmark = pytest.mark.gpu


def ints(mmr, values):
    return mmr.DeviceArray.from_numpy(np.asarray(values, np.int32))


class Forks:
    """Calls on a pool on the device and the same on its host copy."""

    def __init__(self, mmr, pool):
        self.mmr, self.pool = mmr, pool
        self.layers, self.table, self.users = pool.upload(mmr)
        self.error = ints(mmr, [0])
        size = mmr.kv8_fork_workspace_size(pool.seqs, pool.per_seq, pool.pages)
        self.workspace = mmr.DeviceArray.from_numpy(np.full(size, 0xA5, np.uint8))

    def __call__(self, parent, keep, room, sinks=0, window=0, pages=True):
        self.error.zero()
        self.mmr.kv8_fork(self.layers, self.users, ints(self.mmr, parent), ints(self.mmr, keep), ints(self.mmr, room),
                          self.workspace, self.error, sinks=sinks, window=window)
        self.mmr.synchronize()
        error = paging.fork(self.pool, parent, keep, room, sinks, window)
        self.check(pages)
        assert int(self.error.numpy()[0]) == error
        return error

    def check(self, pages=True):
        np.testing.assert_array_equal(self.table.numpy(), self.pool.table)
        np.testing.assert_array_equal(self.users.numpy(), self.pool.users)
        if pages:
            self.pool.assert_pages_equal()


SHAPES = [(1, 1, 32), (3, 2, 96), (2, 4, 64), (2, 1, 128), (70, 1, 32), (1, 64, 32), (1, 21, 64)]  # layers, KV heads, head dimension


@pytest.mark.parametrize("layers,heads,d", SHAPES)
@pytest.mark.parametrize("seed", range(3))
def test_forks_at_random(gpu, layers, heads, d, seed):
    rng = np.random.default_rng(seed * 7 + d + layers)
    seqs = int(rng.integers(1, 9))
    pool = paging.Pool(rng, layers, 60, seqs, 8, heads, d)
    tokens = rng.integers(0, 64 * 8 // 2, seqs)
    pool.fill(rng, tokens, 0.4)
    step = Forks(gpu, pool)
    for i in range(6):
        parent = rng.integers(-1, seqs, seqs)
        keep = np.where(parent >= 0, np.minimum(tokens[parent], rng.integers(0, 600, seqs)), 0)
        room = np.minimum(rng.choice([0, 1, 1, 5, 64, 100], seqs), 64 * 8 - keep)
        sinks, window = (0, 0) if i % 2 else (int(rng.integers(0, 100)), int(rng.integers(1, 300)))
        print(f"[case] {layers},{heads},{d} parent {parent} keep {keep} room {room} {sinks} {window}", flush=True)
        step(parent, keep, room, sinks, window)
        tokens = keep + room


@pytest.mark.parametrize("group,context", [(4, 0), (4, 63), (4, 64), (4, 65), (2, 777), (8, 130), (1, 100)])
def test_beams(gpu, group, context):
    """Searches whose beams go on from each other, token by token over a page's end."""
    rng = np.random.default_rng(group + context)
    seqs, per = 3 * group, context // 64 + 3
    pool = paging.Pool(rng, 2, seqs * per + 5, seqs, per, 2, 64)
    pool.fill(rng, [context] * seqs)
    step = Forks(gpu, pool)
    for i in range(8):
        parent = np.arange(seqs) // group * group + rng.integers(0, group, seqs)
        assert step(parent, [context + i] * seqs, [1] * seqs) == 0


def test_one_prompt_for_all(gpu):
    """A prompt of one sequence, then everyone's; then they part, and end one by one until the pool is free."""
    rng = np.random.default_rng(5)
    seqs = 40
    pool = paging.Pool(rng, 2, 200, seqs, 6, 1, 64)
    step = Forks(gpu, pool)
    step([-1] * seqs, [0] * seqs, [150] + [0] * (seqs - 1))
    step([0] * seqs, [150] * seqs, [0] * seqs)  # shared, nothing is written
    assert (pool.users[pool.table[0, :3]] == seqs).all()
    step(np.arange(seqs), [150] * seqs, [3] * seqs)  # all copy but the first
    assert (pool.users[pool.table[:, 2]] == 1).all()
    for s in range(0, seqs, 13):
        parent = np.where(np.arange(seqs) < s, -1, np.arange(seqs))
        step(parent, np.where(parent < 0, 0, 150), [0] * seqs)
    step([-1] * seqs, [0] * seqs, [0] * seqs)
    assert (pool.users == 0).all() and (pool.table == -1).all()


def test_pages_kept_by_the_caller(gpu):
    """A page that the caller counts too is not written, not freed and not taken."""
    rng = np.random.default_rng(6)
    pool = paging.Pool(rng, 1, 12, 2, 4, 1, 32)
    pool.fill(rng, [100, 0])
    kept = [int(p) for p in pool.table[0, :2]]
    pool.users[kept] += 1
    step = Forks(gpu, pool)
    step([0, -1], [100, 0], [1, 0])  # writing after token 100 takes a copy of the second page
    assert pool.table[0, 0] == kept[0] and pool.table[0, 1] != kept[1]
    step([-1, -1], [0, 0], [0, 256])
    assert (pool.users[kept] == 1).all() and not set(kept) & set(pool.table[1])


def test_a_page_twice_in_a_row(gpu):
    """A row that names a page at two places counts it twice, and copies it before it writes to it."""
    rng = np.random.default_rng(16)
    pool = paging.Pool(rng, 2, 9, 3, 4, 1, 64)
    pool.table[0, :3], pool.table[1, :2] = [5, 2, 5], [7, 7]
    pool.users[[5, 2, 7]] = 2, 1, 2
    step = Forks(gpu, pool)
    step([0, 1, 0], [130, 128, 70], [1, 0, 64])
    assert pool.table[0, 2] not in (5, 2) and pool.users[5] == 2
    step([0, 0, 1], [131, 131, 100], [1, 1, 1])
    step([-1, 1, 1], [0, 50, 50], [0, 2, 2])


def test_most_sequences(gpu):
    rng = np.random.default_rng(17)
    pool = paging.Pool(rng, 1, 3000, 65535, 1, 1, 32)
    step = Forks(gpu, pool)
    room = np.zeros(65535, int)
    room[rng.permutation(65535)[:2500]] = 40
    step([-1] * 65535, np.zeros(65535, int), room)
    holders = np.flatnonzero(pool.table[:, 0] >= 0)
    parent = np.full(65535, -1)
    parent[holders] = rng.permutation(holders)
    parent[rng.permutation(65535)[:300]] = holders[0]
    keep = np.where(parent >= 0, 40, 0)
    step(parent, keep, np.where(parent >= 0, rng.integers(0, 2, 65535), 0))


def test_pools_on_two_streams(gpu):
    """Calls of two pools that run at the same time, each on its stream and workspace."""
    mmr, rng = gpu, np.random.default_rng(18)
    forks, streams, plans = [], [mmr.Stream(), mmr.Stream()], []
    for seqs in (16, 24):
        pool = paging.Pool(rng, 3, 200, seqs, 6, 2, 64)
        pool.fill(rng, [100] * seqs, 0.3)
        forks.append(Forks(mmr, pool))
        plan = rng.integers(0, seqs, seqs), np.full(seqs, 100), np.full(seqs, 30)
        plans.append((plan, [ints(mmr, a) for a in plan]))
    mmr.synchronize()
    for _ in range(20):
        for f, (_, device), stream in zip(forks, plans, streams):
            mmr.kv8_fork(f.layers, f.users, *device, f.workspace, f.error, stream=stream)
    mmr.synchronize()
    for f, (plan, _) in zip(forks, plans):
        for _ in range(20):
            paging.fork(f.pool, *plan)
        f.check()


def test_no_more_pages(gpu):
    rng = np.random.default_rng(7)
    pool = paging.Pool(rng, 2, 6, 4, 5, 1, 64)
    pool.fill(rng, [70, 0, 0, 0])
    step = Forks(gpu, pool)
    assert step([0, 0, -1, -1], [70, 70, 0, 0], [1, 1, 200, 64]) == paging.NO_PAGES
    # The page that is to be copied has no place: what was asked for before it has.
    pool = paging.Pool(rng, 2, 3, 3, 5, 1, 64)
    pool.fill(rng, [70, 0, 0])
    step = Forks(gpu, pool)
    assert step([0, -1, 0], [70, 0, 70], [1, 64, 1]) == paging.NO_PAGES
    assert pool.table[2, 1] == -1
    # All of a table row at once, and a pool that is used to its last page.
    pool = paging.Pool(rng, 1, 5, 1, 5, 1, 32)
    assert Forks(gpu, pool)([-1], [0], [320]) == 0 and (pool.users == 1).all()


def test_fork_refuses_on_the_device(gpu):
    """What cannot be is flagged and its sequence ends; the others are forked."""
    rng = np.random.default_rng(8)
    for bad in ([(6, 0, 0)], [(-2, 0, 0)], [(0, -1, 1)], [(0, 5, -1)], [(0, 100, 221)], [(0, 2 ** 31 - 1, 2 ** 31 - 1)],
                [(-1, 7, 321)]):
        pool = paging.Pool(rng, 1, 30, 6, 5, 1, 32)
        pool.fill(rng, [130, 40, 200, 0, 64, 1], 0.5)
        parent, keep, room = [0, 1, 0, 0, 4, 5], [130, 40, 100, 64, 64, 1], [1, 1, 1, 1, 1, 1]
        parent[2], keep[2], room[2] = bad[0]
        assert Forks(gpu, pool)(parent, keep, room) == paging.BAD_ROWS, bad
    # A partly filled page without a number, and a parent that is nobody with tokens to keep.
    pool = paging.Pool(rng, 1, 30, 3, 5, 1, 32)
    pool.fill(rng, [130, 40, 0])
    pool.users[pool.table[0, 2]] -= 1
    pool.table[0, 2] = 30
    assert Forks(gpu, pool)([0, 1, 0], [130, 40, 70], [1, 1, 0]) == paging.BAD_ROWS
    pool = paging.Pool(rng, 1, 30, 2, 5, 1, 32)
    pool.fill(rng, [130, 40])
    assert Forks(gpu, pool)([-1, 1], [100, 40], [5, 1]) == 0


@pytest.mark.parametrize("seqs,per,pages", [(1200, 5, 9000), (3, 3000, 10000), (2500, 1, 2600)])
def test_many_sequences_and_pages(gpu, seqs, per, pages):
    """More than one pass of the one block over sequences and pages, and table rows of more than one block."""
    rng = np.random.default_rng(seqs)
    pool = paging.Pool(rng, 1, pages, seqs, per, 1, 32)
    tokens = rng.integers(0, 64 * per, seqs)
    pool.fill(rng, tokens, 0.3)
    step = Forks(gpu, pool)
    for _ in range(3):
        parent = rng.integers(0, seqs, seqs)
        keep, room = np.minimum(tokens[parent], 64 * per - 1), np.ones(seqs, int)
        step(parent, keep, room)
        tokens = keep + room


@pytest.mark.parametrize("pages,free", [(16384, 0.1), (16385, 0.1), (18000, 0.001), (19001, 0.3), (20480, 1.0)])
def test_free_pages_of_large_pools(gpu, pages, free):
    """Free pages far apart among those that the caller keeps, more and fewer than are wanted."""
    rng = np.random.default_rng(pages)
    seqs, per = 6, 40
    pool = paging.Pool(rng, 1, pages, seqs, per, 1, 32)
    pool.users[:] = rng.random(pages) >= free
    pool.users[-1] = 0  # the last page is the last to be taken
    step = Forks(gpu, pool)
    wanted = [64 * per, 1, 0, 64 * per, 640, 65]
    error = step([-1] * seqs, [0] * seqs, wanted)
    assert (error == 0) == ((pool.users == 0).any() or free > 0.01)
    tokens = [n if (pool.table[s, : -(-n // 64)] >= 0).all() else 0 for s, n in enumerate(wanted)]
    step([5, 5, 1, -1, 4, 0], [tokens[5], tokens[5] // 2, tokens[1], 0, tokens[4], tokens[0]], [1, 70, 3, 0, 64, 0])
    step([-1] * seqs, [0] * seqs, [64 * per] * seqs)


def test_windows_free_pages(gpu):
    """A chat grows far past its window on a pool of little more pages than that."""
    rng = np.random.default_rng(9)
    pool = paging.Pool(rng, 2, 10, 1, 200, 1, 32)
    step, sinks, window = Forks(gpu, pool), 70, 300
    step([-1], [0], [1])
    for n in range(1, 2000, 37):
        assert step([0], [n], [37], sinks, window) == 0
        held = np.flatnonzero(pool.table[0] >= 0)
        assert set(held) >= {p for p in range(-(-n // 64)) if p < 2 or p * 64 + 63 > n - window}


@pytest.mark.parametrize("layers,heads,d", SHAPES)
@pytest.mark.parametrize("pages,seqs,tokens", [(40, 4, 300), (1, 1, 64), (7, 1, 0), (50, 5, 640), (300, 9, 1500)])
def test_compact(gpu, layers, heads, d, pages, seqs, tokens):
    mmr, rng = gpu, np.random.default_rng(pages + d)
    pool = paging.Pool(rng, layers, pages, seqs, 25, heads, d)
    pool.fill(rng, [tokens] + [int(n) for n in rng.integers(0, tokens + 1, seqs - 1)], 0.3)
    pool.table[-1, -1] = pages  # no page
    for alias in (False, True):
        layer_refs, table, users = pool.upload(mmr)
        was_table, was_users = pool.table.copy(), pool.users.copy()
        out = (table, users) if alias else (ints(mmr, was_table * 0 + 99), ints(mmr, was_users * 0 + 99))
        moved, live = ints(mmr, [77] * pages), ints(mmr, [0])
        size = mmr.kv8_compact_workspace_size(pages)
        mmr.kv8_compact(layer_refs, users, *out, moved, live, mmr.DeviceArray(size, np.uint8))
        mmr.synchronize()
        saved = [getattr(pool, n).copy() for n in pool.NAMES]
        want_moved, want_live = paging.compact(pool)
        assert int(live.numpy()[0]) == want_live
        np.testing.assert_array_equal(moved.numpy(), want_moved)
        np.testing.assert_array_equal(out[0].numpy(), pool.table)
        np.testing.assert_array_equal(out[1].numpy(), pool.users)
        pool.assert_pages_equal()
        assert (pool.users[:want_live] > 0).all() and (pool.users[want_live:] == 0).all()
        if not alias:
            np.testing.assert_array_equal(table.numpy(), was_table)
            np.testing.assert_array_equal(users.numpy(), was_users)
            pool.table, pool.users = was_table, was_users
            for n, a in zip(pool.NAMES, saved):
                setattr(pool, n, a)


@pytest.mark.parametrize("alias", [True, False])
@pytest.mark.parametrize("pages,part", [(20000, 0.5), (5000, 0.02), (5000, 0.97), (4097, 1.0), (9000, 0.0), (16384, 0.6),
                                        (16385, 0.6), (17000, 1.0), (17408, 0.0), (18433, 0.9999), (16400, 0.0001)])
def test_compact_many_pages(gpu, pages, part, alias):
    mmr, rng = gpu, np.random.default_rng(pages)
    pool = paging.Pool(rng, 1, pages, 10, pages // 10 + 1, 1, 32)
    used = rng.permutation(pages)[: int(pages * part)]
    flat = pool.table.reshape(-1)
    flat[rng.permutation(flat.size)[: used.size]] = used
    pool.users[used] = rng.integers(1, 4, used.size)  # the caller's own among them
    layer_refs, table, users = pool.upload(mmr)
    moved, live = ints(mmr, [77] * pages), ints(mmr, [0])
    workspace = mmr.DeviceArray.from_numpy(np.full(mmr.kv8_compact_workspace_size(pages), 0xA5, np.uint8))
    was_users, source = pool.users.copy(), users
    if not alias:
        table, users = ints(mmr, pool.table * 0 + 99), ints(mmr, pool.users * 0 + 99)
    mmr.kv8_compact(layer_refs, source, table, users, moved, live, workspace)
    mmr.synchronize()
    if not alias:
        np.testing.assert_array_equal(source.numpy(), was_users)
    want_moved, want_live = paging.compact(pool)
    assert int(live.numpy()[0]) == want_live
    np.testing.assert_array_equal(moved.numpy(), want_moved)
    np.testing.assert_array_equal(table.numpy(), pool.table)
    np.testing.assert_array_equal(users.numpy(), pool.users)
    pool.assert_pages_equal()


def test_pages_past_four_gigabytes(gpu):
    """Copies and moves between page numbers whose offsets take more than 32 bits."""
    mmr, rng = gpu, np.random.default_rng(11)
    heads, d, pages = 2, 128, 300_000  # 4.9 GB of codes each
    nbytes, ebytes = heads * 64 * d, heads * 4
    buffers = [mmr.DeviceArray((pages, n), np.int8) for n in (nbytes, nbytes, ebytes, ebytes)]
    users = np.ones(pages, np.int32)
    users[[5, 250_000, 299_999]] = 0
    table = ints(mmr, np.full((2, 4), -1))
    layer = mmr.Kv8Layers([mmr.Kv8Pages(*buffers, table, pages, 2, 4, heads, d)])
    d_users, error = ints(mmr, users), ints(mmr, [0])

    def put(page):
        out = []
        for b in buffers:
            a = rng.integers(-128, 128, b.shape[1]).astype(np.int8)
            mmr.check(mmr.lib().mmr_memcpy_h2d(b.ptr + page * b.shape[1], a.ctypes.data, a.nbytes))
            out.append(a)
        return out

    def get(page):
        out = [np.empty(b.shape[1], np.int8) for b in buffers]
        for a, b in zip(out, buffers):
            mmr.check(mmr.lib().mmr_memcpy_d2h(a.ctypes.data, b.ptr + page * b.shape[1], a.nbytes))
        return out

    old = put(299_998)
    table.upload(np.array([[299_998, -1, -1, -1], [299_998, -1, -1, -1]], np.int32))
    users[299_998] = 2
    d_users.upload(users)
    workspace = mmr.DeviceArray(mmr.kv8_fork_workspace_size(2, 4, pages), np.uint8)
    before = get(5)
    # Both grow past token 40: the second copies to the lowest free page.
    mmr.kv8_fork(layer, d_users, ints(mmr, [0, 1]), ints(mmr, [40, 40]), ints(mmr, [25, 1]), workspace, error)
    mmr.synchronize()
    np.testing.assert_array_equal(table.numpy(), [[299_998, 5, -1, -1], [250_000, -1, -1, -1]])
    assert int(error.numpy()[0]) == 0
    now = get(250_000)
    keys, was = now[0].reshape(heads, 64, d), old[0].reshape(heads, 64, d)
    np.testing.assert_array_equal(keys[:, :48], was[:, :48])
    values, was = now[1].reshape(heads, d, 64), old[1].reshape(heads, d, 64)
    np.testing.assert_array_equal(values[..., :48], was[..., :48])
    for a, b in zip(now[2:], old[2:]):
        np.testing.assert_array_equal(a.reshape(heads, 4)[:, :3], b.reshape(heads, 4)[:, :3])
    np.testing.assert_array_equal(get(5)[0], before[0])
    # Of the last pages, one moves into a hole that is far, too.
    users = d_users.numpy()
    assert users[299_999] == 0
    users[[260_000, 299_997]] = 0
    d_users.upload(users)
    mmr.kv8_compact(layer, d_users, table, d_users, ints(mmr, np.zeros(pages)), ints(mmr, [0]),
                    mmr.DeviceArray(mmr.kv8_compact_workspace_size(pages), np.uint8))
    mmr.synchronize()
    np.testing.assert_array_equal(table.numpy(), [[260_000, 5, -1, -1], [250_000, -1, -1, -1]])
    for a, b in zip(get(260_000), old):
        np.testing.assert_array_equal(a, b)


def test_recorded_forks_share_a_workspace(gpu):
    """Two recorded calls on one workspace and an eager one between, on pools of their own."""
    mmr, rng = gpu, np.random.default_rng(13)
    stream, forks, graphs = mmr.Stream(), [], []
    for seqs in (8, 3):
        pool = paging.Pool(rng, 2, 80, seqs, 6, 1, 64)
        pool.fill(rng, rng.integers(0, 200, seqs), 0.3)
        forks.append(Forks(mmr, pool))
    workspace = max((f.workspace for f in forks), key=lambda w: w.nbytes)
    args = []
    for f in forks:
        n = f.pool.seqs
        plan = rng.integers(0, n, n), np.full(n, 70), np.full(n, 60)
        f([0] * n, [100] * n, [40] * n)  # all have tokens to keep
        device = [ints(mmr, a) for a in plan]
        args.append((plan, device))
        with mmr.Graph(stream) as graph:
            mmr.kv8_fork(f.layers, f.users, *device, workspace, f.error, stream=stream)
        graphs.append(graph)
        mmr.synchronize()
        f.check()  # recording ran nothing
    for i in (0, 1, 1, 0, 0, 1):
        graphs[i].launch(stream)
        mmr.synchronize()
        paging.fork(forks[i].pool, *args[i][0])
        forks[i].check()
        other = forks[1 - i]
        mmr.kv8_fork(other.layers, other.users, *args[1 - i][1], workspace, other.error, stream=stream)
        mmr.synchronize()
        paging.fork(other.pool, *args[1 - i][0])
        other.check()
