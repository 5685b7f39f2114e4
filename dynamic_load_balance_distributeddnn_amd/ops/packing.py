"""Packed sequences and distance buckets, shared by the long-context ops.

Both are plain host-side descriptions; nothing here reads a device.
"""

from __future__ import annotations

import math
from functools import cached_property, lru_cache

import numpy as np
import torch

# Rows of a sequence one workgroup of the attention kernels owns
# (PA_ROWS in csrc/packed_attn.h).
TILE_ROWS = 128
# Workgroups a launch takes: below 2**32 threads, 256 each.
MAX_WORKGROUPS = 2 ** 24 - 1


class PackedSequences:
    """Sequences of the given lengths, packed behind each other.

    Sequence ``s`` owns the rows ``offsets[s]`` to ``offsets[s + 1]`` of
    every packed tensor; rows from ``total`` on belong to none.  Lengths
    are host integers (zero is allowed), so they are checked here once and
    no kernel reads a length that nobody looked at.  Build one per batch
    and use it for all layers, forward and backward, on any stream; it has
    to outlive a captured graph that used it.  With a ``device`` it is for
    tensors of that device only.

    For each head layout it is used with it keeps work lists on the device,
    of the query tiles and, for gradients, of the key tiles.  A list's tiles
    times the heads have to be below 2**24 (2**20 sequences of one row with
    16 heads are too many).
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
        if sum(n.tolist()) >= 2 ** 30:  # whole numbers of any size
            raise ValueError("more than 2**30 - 1 rows in one packing")
        self._n = n
        self.lengths = tuple(n.tolist())
        self.offsets = (0, *np.cumsum(n).tolist())
        self.total = self.offsets[-1]
        self.device = None if device is None else torch.device(device)
        self._lists = {}

    def __len__(self):
        return len(self.lengths)

    @cached_property
    def _tiles(self):
        """(sequence, tile) of every 128-row tile."""
        tiles = -(-self._n // TILE_ROWS)
        seq = np.repeat(np.arange(len(tiles)), tiles)
        return seq, np.arange(len(seq)) - (np.cumsum(tiles) - tiles)[seq]

    def host_work(self, heads, kv_heads, rows=32, at_once=512):
        """((list, chunks, slots) of the query tiles, of the key tiles)."""
        return (self._query_work(heads),
                self._key_work(heads, kv_heads, rows, at_once))

    def _query_work(self, heads):
        """A query tile reads the 64-key tiles up to its last row.  Tiles
        with much more to do than a workgroup's share of the whole are cut
        into chunks, whose sums a second kernel joins."""
        seq, tile = self._tiles
        steps = -(-np.minimum((tile + 1) * TILE_ROWS, self._n[seq]) // 64)
        total = int(steps.sum()) * heads
        # The longest tile is what a launch takes at least.  The limits count
        # on 512 workgroups at a time, which is right for heads of over 64;
        # of smaller ones 768 to 1024 fit, and places stay empty: one of 4001,
        # 12 heads of 64 with a bias, is 576 chunks and takes as long as the
        # longest.  Cutting costs a trip of the sums through memory:
        # one sequence of 4001, 12 heads of 64, forward 73 -> 50 us where
        # the longest is 2.7 times a place's share, but seven packed ones,
        # 16 heads of 128 over 4, 79 -> 85 where it is 1.3 times, and six of
        # 1024, 12 heads of 64, 26 -> 30 where it is 1.6 times.  Chunks of
        # a 384th, the unequal ones then fill the places: five of 4096 in
        # all, 16 heads of 128, 46 us, with a 512th 50, a 768th 53.
        limit = max(8, total // 384)
        if len(steps) and int(steps.max()) <= 1.75 * total / 512:
            limit = int(steps.max())
        return self._chunks(seq, tile, steps, heads, limit)

    def _key_work(self, heads, kv_heads, rows, at_once):
        """A key tile is read by the tiles of ``rows`` queries from its
        first row on, of every head that shares it; ``at_once`` workgroups
        run at a time.

        These are longer and more uneven, and how well the chunks of a
        limit fill the places decides: the limit is the best of a few by
        what their launch and join take, in steps.  A chunk costs 8 of its
        own, a join 2.5 and 0.012 each chunk and head (measured, 1.2 to 2
        us a step; all for steps of 32 rows).  Backward in us, with limits
        of a share of the whole by 384, 512, 640 and 768, and the one taken:
        one of 8192, 16 heads of 64 over 4, 621, 572, 560, 623 (640); five
        of 4096 in all, 16 heads of 64 with a bias, 114, 118, 126, 125
        (384); one of 8192, 32 heads of 128 over 8, 2109, 2040, 1968, 1912
        (768).  Below 12 steps chunks lose: eight of 512, 16 heads of 128
        over 4, 102 us with 8, 91 with 12, 98 with 16.
        """
        seq, tile = self._tiles
        steps = (-(-(self._n[seq] - tile * TILE_ROWS) // rows)
                 * (heads // kv_heads))
        longest = int(steps.max()) if len(steps) else 0
        total = int(steps.sum()) * kv_heads
        least = 12 * 32 // rows
        # many tiles a place: nothing to gain by cutting
        if 2 * longest * at_once <= total or longest <= least:
            return self._chunks(seq, tile, steps, kv_heads, longest)
        limits = {max(least, total // n) for n in (384, 512, 640, 768)}
        limit = min(sorted(limits | {longest}),
                    key=lambda x: self._time(steps, kv_heads, x, at_once,
                                             32 / rows))
        return self._chunks(seq, tile, steps, kv_heads, limit)

    @staticmethod
    def _time(steps, heads, limit, at_once, unit):
        parts = -(-steps // limit)
        sizes = np.sort(np.repeat(steps / parts, parts * heads))[::-1]
        sizes = sizes + 8 * unit
        # the longest first, each to the place that is free first
        load = np.zeros(at_once)
        for i in range(0, len(sizes), at_once):
            part = sizes[i:i + at_once]
            load[:len(part)] += part
            load.sort()
        slots = int((parts * (parts > 1)).sum()) * heads
        return load[-1] + ((2.5 + 0.012 * slots) * unit if slots else 0.0)

    def _chunks(self, seq, tile, steps, heads, limit):
        """Chunks of at most ``limit`` steps, the longest first, then the
        joins of the tiles that are in several; a workgroup a chunk and
        head."""
        parts = -(-steps // max(limit, 1))
        if int(parts.sum()) * heads > MAX_WORKGROUPS:
            raise ValueError(f"{int(parts.sum())} tiles of {heads} heads are "
                             "too many for one launch, 2**24 - 1 in all: use "
                             "several packings")
        first = np.asarray(self.offsets[:-1], np.int64)[seq]
        if not len(steps) or int(steps.max()) <= limit:
            order = np.argsort(-steps, kind="stable")
            rows = np.zeros((len(steps), 8), np.int32)
            rows[:, 0] = first[order]
            rows[:, 1] = self._n[seq[order]]
            rows[:, 2] = tile[order]
            rows[:, 4] = steps[order]
            rows[:, 5] = -1
            return rows, len(rows), 0
        which = np.repeat(np.arange(len(steps)), parts)
        part = np.arange(len(which)) - (np.cumsum(parts) - parts)[which]
        cut = parts > 1
        slots = np.cumsum(parts * cut) - parts * cut
        rows = np.zeros((len(which) + int(cut.sum()), 8), np.int32)
        chunks, joins = rows[:len(which)], rows[len(which):]
        chunks[:, 0] = first[which]
        chunks[:, 1] = self._n[seq[which]]
        chunks[:, 2] = tile[which]
        chunks[:, 3] = part * steps[which] // parts[which]
        chunks[:, 4] = (part + 1) * steps[which] // parts[which]
        chunks[:, 5] = np.where(cut[which], slots[which] + part, -1)
        chunks[:] = chunks[np.argsort(chunks[:, 3] - chunks[:, 4],
                                      kind="stable")]
        joins[:, 0] = first[cut]
        joins[:, 1] = self._n[seq[cut]]
        joins[:, 2] = tile[cut]
        joins[:, 3] = slots[cut]
        joins[:, 4] = parts[cut]
        return rows, len(which), int((parts * cut).sum())

    def check_device(self, device):
        own = self.device
        if own is not None and (own.type != device.type or
                                own.index not in (None, device.index)):
            raise ValueError(f"the PackedSequences is for {own}, the "
                             f"tensors are on {device}")

    def query_work(self, device, heads):
        """The query tiles' work list on a device, made at its first use
        (not within a graph capture) and kept."""
        key = (device, heads)
        if key not in self._lists:
            self._lists[key] = self._put(device, self._query_work, heads)
        return self._lists[key]

    def key_work(self, device, heads, kv_heads, rows, at_once):
        """The key tiles', as ``query_work``; only a backward reads it."""
        key = (device, heads, kv_heads, rows, at_once)
        if key not in self._lists:
            self._lists[key] = self._put(device, self._key_work, heads,
                                         kv_heads, rows, at_once)
        return self._lists[key]

    def _put(self, device, make, *args):
        self.check_device(device)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("use the PackedSequences once in this way "
                               "before the capture")
        rows, chunks, slots = make(*args)
        # a synchronous copy: the list is there for every stream
        return torch.from_numpy(rows).to(device), chunks, slots


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
