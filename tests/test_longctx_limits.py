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
