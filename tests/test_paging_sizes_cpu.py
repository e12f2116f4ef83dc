"""Sizes that no launch takes are refused on the host (no GPU needed)."""
from __future__ import annotations

import pytest

from test_low_bit_cpu import At


@pytest.mark.parametrize("searches,beams,vocab", [(65000, 8, 131073), (65536 // 4, 32, 131072), (65535, 8, 131072)])
def test_selections_of_more_blocks_than_a_launch_has(mmr, searches, beams, vocab):
    """Rows of several runs of 4,096 columns take a block of 256 threads a run; a launch has less than 2^32 threads."""
    runs = -(-vocab // 4096)
    if searches * beams * runs * 256 < 2 ** 32:
        assert mmr.beam_select_workspace_size(searches, beams, vocab) > 0
        return
    assert mmr.beam_select_workspace_size(searches, beams, vocab) == 0
    b = At()
    beam = mmr.Beams(b, b, b)
    with pytest.raises(mmr.InvalidArgument, match="too many logits"):
        mmr.beam_select(b, searches, beams, vocab, -1, 0.0, beam, beam, b, b, At(4096, 1 << 60), b)
