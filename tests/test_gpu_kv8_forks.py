"""Forks whose plans leave something open: sequences without a parent that had tokens, counts beside the plans in memory,
pools that run out, and searches that run out of candidates."""
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
