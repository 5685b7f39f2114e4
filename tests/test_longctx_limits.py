"""Limits of packed attention that are checked on the host (CPU)."""

import numpy as np
import pytest
import torch

from dynamic_load_balance_distributeddnn_amd.ops import functional as FD


@pytest.mark.parametrize("lengths", [
    [2 ** 62] * 4, [2 ** 63 - 1, 2 ** 63 - 1, 2], [2 ** 30 - 1, 1],
    np.array([2 ** 64 - 1], np.uint64), torch.tensor([2 ** 62] * 4)])
def test_lengths_whose_sum_leaves_64_bits(lengths):
    """A sum that comes round to a small number is no small packing."""
    with pytest.raises(ValueError):
        FD.PackedSequences(lengths)


def test_the_most_rows():
    assert FD.PackedSequences([2 ** 30 - 2, 0, 1]).total == 2 ** 30 - 1


def test_more_tiles_than_a_launch_takes():
    """2**32 threads are one too many: workgroups of 256, one a tile and
    head."""
    pack = FD.PackedSequences(np.ones(2 ** 20, np.int64))
    with pytest.raises(ValueError, match="too many"):
        pack.host_work(16, 16)
    with pytest.raises(ValueError, match="too many"):
        pack.host_work(32, 8)  # the query tiles alone
    for rows, chunks, slots in pack.host_work(15, 15):
        assert rows.shape == (2 ** 20, 8)
        assert (chunks, slots) == (2 ** 20, 0)


@pytest.mark.parametrize("buckets", [0, 8])
def test_autocast_leaves_the_statistics_in_32_bits(buckets):
    """The composition's own products are not cast on the CPU."""
    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(70, 2, 16, generator=gen) for _ in range(3))
    table = torch.randn(buckets, 2, generator=gen) if buckets else None
    pack = FD.PackedSequences([60, 10])
    for dtype in (torch.float32, torch.bfloat16):
        given = [t.to(dtype) for t in (q, k, v)]
        want = FD.packed_causal_attention(*given, pack, bias_table=table,
                                          max_distance=20)
        with torch.autocast("cpu", dtype=torch.bfloat16):
            got = FD.packed_causal_attention(*given, pack, bias_table=table,
                                             max_distance=20)
        assert got.dtype == dtype and torch.equal(got, want)
