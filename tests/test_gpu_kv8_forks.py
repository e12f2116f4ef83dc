"""Forks whose plans leave something open: sequences without a parent that had tokens, pools that run out, and counts
beside the plans in memory."""
from __future__ import annotations

import numpy as np
import pytest

import paging_reference as paging
from test_gpu_kv8_pages import Forks, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,per", [(4, 5), (300, 5)])  # counted by the deciding block, and by a kernel of its own
def test_keep_of_nobody_counts_as_nothing(gpu, seqs, per):
    """A sequence that ends, or begins anew, may still have its tokens as keep, or anything."""
    rng = np.random.default_rng(21)
    pool = paging.Pool(rng, 1, 8 * seqs, seqs, per, 1, 32)
    pool.fill(rng, rng.integers(0, 200, seqs), 0.3)
    step = Forks(gpu, pool)
    parent, keep, room = np.full(seqs, -1), rng.integers(0, 64 * per, seqs), np.full(seqs, 64 * per)
    keep[:4], room[:4] = [300, 40, -3, 2 ** 31 - 1], [100, 1, 0, 5]
    parent[1] = 1
    step.error.zero()
    gpu.kv8_fork(step.layers, step.users, *(ints(gpu, a) for a in (parent, keep, room)), step.workspace, step.error)
    gpu.synchronize()
    assert paging.fork(pool, parent, np.where(parent < 0, 0, keep), room) == 0
    step.check()
    assert int(step.error.numpy()[0]) == 0


def test_again_after_a_full_pool(gpu):
    """A copy that gets no page takes its kept tokens along.  With table and users put back, and less to keep, the same
    forks have all that the failed call was to keep, though its copies went to pages that it had freed."""
    mmr, rng = gpu, np.random.default_rng(22)
    pool = paging.Pool(rng, 2, 8, 6, 3, 1, 64)
    tokens = [70, 0, 0, 0, 100, 128]  # 2 + 2 + 2 pages, two are free
    pool.fill(rng, tokens)
    step = Forks(mmr, pool)
    was_table, was_users = pool.table.copy(), pool.users.copy()
    was = {n: getattr(pool, n).copy() for n in pool.NAMES}
    # Four go on from the first (three copies), the fifth is taken back by a page, the last begins anew.
    plan = [0, 0, 0, 0, 4, -1], [70, 70, 70, 70, 64, 0], [1, 1, 1, 1, 0, 192]
    assert step(*plan) == paging.NO_PAGES
    assert (pool.table[1:4, 1] >= 0).all() and pool.table[5, 2] == -1
    assert set(pool.table[1:4, 1]) & set(was_table[4:, :2].reshape(-1))  # copies to what was freed
    for room in ([1, 1, 1, 1, 0, 0], [0, 0, 0, 0, 0, 0]):
        step.table.upload(was_table), step.users.upload(was_users)
        pool.table, pool.users[:] = was_table.copy(), was_users
        assert step(*plan[:2], room) == 0
        for s, n in enumerate((70, 70, 70, 70, 64)):
            for t in range(n):
                page, old = pool.table[s, t // 64], was_table[plan[0][s], t // 64]
                np.testing.assert_array_equal(pool.keys[:, page, :, t % 64], was["keys"][:, old, :, t % 64])
                np.testing.assert_array_equal(pool.values[:, page, :, :, t % 64], was["values"][:, old, :, :, t % 64])
    # Without that: of three that copy, the last has no page, and no tokens from 64 on.
    pool = paging.Pool(rng, 2, 4, 4, 3, 1, 64)
    pool.fill(rng, [70, 0, 0, 0])
    step = Forks(mmr, pool)
    assert step([0, 0, 0, 0], [70] * 4, [1] * 4) == paging.NO_PAGES
    np.testing.assert_array_equal(pool.table[:, 1] >= 0, [True, True, True, False])
    assert (pool.table[:, 0] == pool.table[0, 0]).all()


class Part:
    """Some words of a device array, as a call takes them."""

    def __init__(self, array, first):
        self.array, self.first, self.ptr = array, first, array.ptr + 4 * first

    def numpy(self, n):
        return self.array.numpy()[self.first: self.first + n]


@pytest.mark.parametrize("seqs,per", [(4, 5), (4, 400)])  # counted by the deciding block, and by a kernel of its own
def test_plans_counts_and_table_side_by_side(gpu, seqs, per):
    """What a call reads once and what it counts in, in the same lines of memory: counts are read as counted."""
    mmr, rng = gpu, np.random.default_rng(24)
    pool = paging.Pool(rng, 1, 24, seqs, per, 1, 32)
    pool.fill(rng, [200, 130, 64, 31], 0.5)
    _, table, users = pool.upload(mmr)
    plans = [([1, 1, 0, 3], [70, 130, 200, 31], [1, 1, 60, 2]), ([2, 0, -1, 2], [100, 5, 9, 260], [30, 1, 90, 0]),
             ([0, 0, 0, 0], [120] * 4, [5, 0, 9, 1]), ([-1, 1, 3, 0], [120, 120, 0, 125], [0, 10, 0, 3])]
    words = np.concatenate([np.zeros(3 * seqs), pool.users, [0, 0, 0, 0], pool.table.reshape(-1)])
    memory = ints(mmr, words)
    at = 3 * seqs
    parent, keep, room = (Part(memory, i * seqs) for i in range(3))
    users, error, table = Part(memory, at), Part(memory, at + 24), Part(memory, at + 28)
    pages = mmr.Kv8Pages(*pool.device[0], table, 24, seqs, per, 1, 32)
    workspace = mmr.DeviceArray(mmr.kv8_fork_workspace_size(seqs, per, 24), np.uint8)
    for plan in plans:
        words = memory.numpy()
        words[:at] = np.concatenate(plan)
        memory.upload(words)
        mmr.kv8_fork(mmr.Kv8Layers([pages]), users, parent, keep, room, workspace, error)
        mmr.synchronize()
        nobody = np.where(np.asarray(plan[0]) < 0, 0, plan[1])
        assert paging.fork(pool, plan[0], nobody, plan[2]) == 0
        np.testing.assert_array_equal(table.numpy(seqs * per).reshape(seqs, per), pool.table)
        np.testing.assert_array_equal(users.numpy(24), pool.users)
        np.testing.assert_array_equal(memory.numpy()[:at], np.concatenate(plan))
        assert error.numpy(1)[0] == 0
        pool.assert_pages_equal()
