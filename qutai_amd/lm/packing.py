"""Sequences of different lengths laid one behind the other in one row of
tokens: what attention and positions need to keep them apart."""
from __future__ import annotations

from array import array
from bisect import bisect_right
from itertools import accumulate

from ..backends import amd
from ..backends.amd_runtime import get_runtime


class Packing:
    """``lengths``: the tokens of every sequence (0 allowed), in the order in
    which they lie; ``total``: the row's tokens, the sum of lengths unless rows
    behind the last sequence belong to none.  Made once for a batch and used by
    every layer: ``positions`` (int64, device) holds each token's place in its
    sequence, 0 behind the last one."""

    def __init__(self, lengths, total=None):
        lengths = tuple(lengths)
        if any(type(n) is not int or n < 0 for n in lengths):
            raise ValueError("packed sequences have lengths of 0 or more")
        self.lengths = lengths
        self.starts = tuple(accumulate(lengths, initial=0))[:-1]
        self.used = self.starts[-1] + lengths[-1] if lengths else 0
        self.total = self.used if total is None else total
        if type(self.total) is not int or self.total < self.used or self.total >= 1 << 31:
            raise ValueError("total is at least the sum of lengths, below 2^31")
        self.longest = max(lengths, default=0)
        self.extent = self.used, len(lengths), self.longest  # what the kernels' shapes are chosen by
        self._positions, self._tiles, self._plans = None, {}, {}

    @property
    def positions(self):
        if self._positions is None:
            positions = amd.AMDStorage(self.total, "int64")
            if self.total:
                starts = amd.storage(array("q", self.starts), dtype="int64")
                positions.runtime.call("qutai_amd_positions", starts.ptr, len(self.starts), self.used, self.total,
                                       positions.ptr)
            self._positions = positions
        return self._positions

    def plan(self, number, heads, kv_heads, dim, dtype, whole, scale, causal):
        """(tiles, count, rows of a tile, bytes of workspace) of pass ``number`` of
        attention (forward, queries of the backward, its keys) of these sizes; asked of
        the library once."""
        key = number, heads, kv_heads, dim, dtype, whole, scale, bool(causal)
        found = self._plans.get(key)
        if found is None:
            lib, sizes = get_runtime().lib, (heads, kv_heads, dim, dtype)
            rows = lib.qutai_amd_attention_packed_rows(*self.extent, *sizes, int(whole), scale, number)
            need = lib.qutai_amd_attention_packed_workspace(*self.extent[:2], *sizes, rows) if number == 2 else 0
            found = (*self.tiles(rows, "length" if not causal else "start" if number == 2 else "end"), rows, need)
            self._plans[key] = found
        return found

    def tiles(self, rows, longest_first):
        """(storage, count): the tiles of ``rows`` tokens of a sequence that the
        workgroups of attention take: an int64 for each that holds the sequence's
        start and, 32 bits up, the tile's first token in it, then as many of the
        sequences' lengths.  Tiles that have most to do come first, by whole tiles:
        causal queries see what lies before them (``longest_first`` "end"), causal
        keys are seen by what lies behind ("start"), and without a mask the work
        goes by the length ("length")."""
        key = rows, longest_first
        if key not in self._tiles:
            order = sorted((i for i, n in enumerate(self.lengths) if n), key=self.lengths.__getitem__, reverse=True)
            lengths = array("q", map(self.lengths.__getitem__, order))
            starts = [self.starts[i] for i in order]
            words, sizes, shift = [], array("q"), rows << 32
            if longest_first == "length":
                for start, n in zip(starts, lengths):
                    count = -(-n // rows)
                    words += range(start, start + count * shift, shift)
                    sizes.extend([n] * count)
            else:  # the sequences of more than `level` tiles are the first ones
                if longest_first == "start":  # their tiles counted from the last
                    starts, shift = [s + (n - 1) // rows * shift for s, n in zip(starts, lengths)], -shift
                rising = lengths[::-1]
                for level in range((self.longest - 1) // rows, -1, -1):
                    many, first = len(lengths) - bisect_right(rising, level * rows), level * shift
                    words += [s + first for s in starts[:many]]
                    sizes += lengths[:many]
            self._tiles[key] = amd.storage(array("q", words) + sizes, dtype="int64"), len(words)
        return self._tiles[key]
