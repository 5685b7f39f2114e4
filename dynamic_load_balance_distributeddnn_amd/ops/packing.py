"""Packed sequences and distance buckets, shared by the long-context ops.

Both are plain host-side descriptions; nothing here reads a device.
"""

from __future__ import annotations

import math
from functools import lru_cache

import numpy as np
import torch

# Rows of a sequence one workgroup of the attention kernels owns
# (PA_ROWS in csrc/packed_attn.h).
TILE_ROWS = 128


class PackedSequences:
    """Sequences of the given lengths, packed behind each other.

    Sequence ``s`` owns the rows ``offsets[s]`` to ``offsets[s + 1]`` of
    every packed tensor; rows from ``total`` on belong to none.  Lengths
    are host integers (zero is allowed), so they are checked here once and
    no kernel reads a length that nobody looked at.  Build one per batch
    and use it for all layers, forward and backward, on any stream; it has
    to outlive a captured graph that used it.

    On the device it keeps two work lists of 128-row tiles, the ones with
    most to do first: for the queries (a tile reads the keys up to its
    last row) and for the keys (a tile is read by the rows from its first
    on).
    """

    def __init__(self, lengths, device=None):
        if isinstance(lengths, torch.Tensor):
            if lengths.is_cuda:
                raise TypeError("PackedSequences wants host lengths; a copy "
                                "from the GPU would wait for it")
            if lengths.is_floating_point() or lengths.dtype == torch.bool:
                raise TypeError("lengths have to be whole numbers")
            lengths = lengths.tolist()
        n = np.asarray(lengths if len(lengths) else np.zeros(0, np.int64))
        if n.ndim != 1 or not np.issubdtype(n.dtype, np.integer):
            raise TypeError("lengths have to be a list of whole numbers")
        n = n.astype(np.int64)
        if (n < 0).any():
            raise ValueError("lengths must not be negative")
        if int(n.sum()) >= 2 ** 30:
            raise ValueError("more than 2**30 - 1 rows in one packing")
        self._n = n
        self.lengths = tuple(n.tolist())
        self.offsets = (0, *np.cumsum(n).tolist())
        self.total = self.offsets[-1]
        self._tables = {}
        if device is not None and torch.device(device).type == "cuda":
            self.tables(device)

    def __len__(self):
        return len(self.lengths)

    def _host_tables(self):
        n = self._n
        tiles = -(-n // TILE_ROWS)
        seq = np.repeat(np.arange(len(n)), tiles)
        first_tile = np.cumsum(tiles) - tiles
        tile = np.arange(len(seq)) - first_tile[seq]
        items = np.zeros((len(seq), 4), np.int32)
        items[:, 0] = np.asarray(self.offsets[:-1], np.int64)[seq]
        items[:, 1] = n[seq]
        items[:, 2] = tile
        seen = np.minimum((tile + 1) * TILE_ROWS, n[seq])
        seeing = n[seq] - tile * TILE_ROWS
        return np.stack([items[np.argsort(-seen, kind="stable")],
                         items[np.argsort(-seeing, kind="stable")]])

    def tables(self, device):
        """(query tiles, key tiles), int32 [tiles, 4] each: the sequence's
        first row, its length, the tile, unused."""
        device = torch.device(device)
        if device.index is None:
            device = torch.device(device.type, torch.cuda.current_device())
        if device not in self._tables:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("build the PackedSequences for its device "
                                   "before the capture")
            # a synchronous copy: the tables are there for every stream
            both = torch.from_numpy(self._host_tables()).to(device)
            self._tables[device] = (
                both, torch.cuda.current_stream(device))
        both, made_on = self._tables[device]
        now = torch.cuda.current_stream(device)
        if now != made_on:
            both.record_stream(now)
        return both[0], both[1]


@lru_cache(maxsize=64)
def bucket_starts(side: int, max_distance: int) -> tuple[int, ...]:
    """Least distance of each of ``side`` buckets.

    The first ``e = side // 2`` buckets hold one distance each.  The other
    ``L = side - e`` divide the logarithm from e to ``max_distance``
    evenly: bucket e + t starts at the least n with
    n >= e * (max_distance / e) ** (t / L), found in whole numbers
    (n**L >= max_distance**t * e**(L - t)), so no rounding moves a border.
    Everything from the last start on, however far, is the last bucket.
    """
    e = side // 2
    steps = side - e
    starts = list(range(e + 1))
    for t in range(1, steps):
        goal = max_distance ** t * e ** (steps - t)
        # at most one off in floating point; settled in whole numbers
        n = int(e * math.exp(math.log(max_distance / e) * t / steps))
        while n ** steps >= goal:
            n -= 1
        while n ** steps < goal:
            n += 1
        starts.append(n)
    return tuple(starts)


def checked_starts(num_buckets: int, max_distance: int,
                   bidirectional: bool) -> tuple[int, ...]:
    """``bucket_starts`` of one side, with the arguments' checks."""
    if not 2 <= num_buckets <= 256:
        raise ValueError(f"2 to 256 buckets are supported, got {num_buckets}")
    if bidirectional and (num_buckets % 2 or num_buckets < 4):
        raise ValueError("a bidirectional bias wants an even number of "
                         f"buckets, 4 at least, got {num_buckets}")
    side = num_buckets // 2 if bidirectional else num_buckets
    max_distance = int(max_distance)
    if not side // 2 < max_distance < 2 ** 30:
        raise ValueError(
            f"max_distance has to be over {side // 2} (the distances with a "
            f"bucket of their own) and below 2**30, got {max_distance}")
    return bucket_starts(side, max_distance)
