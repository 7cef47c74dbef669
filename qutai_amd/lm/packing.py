"""Sequences of different lengths laid one behind the other in one row of
tokens: what attention and positions need to keep them apart."""
from __future__ import annotations

from array import array
from itertools import accumulate, chain

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
            places = array("q", chain.from_iterable(map(range, self.lengths)))
            places.extend([0] * (self.total - self.used))
            self._positions = amd.storage(places, dtype="int64")
        return self._positions

    def plan(self, number, heads, kv_heads, dim, dtype, whole, scale, causal):
        """(tiles, count, rows of a tile) of pass ``number`` of attention (forward,
        queries of the backward, its keys) of these sizes; asked of the library once."""
        key = number, heads, kv_heads, dim, dtype, whole, scale, bool(causal)
        found = self._plans.get(key)
        if found is None:
            rows = get_runtime().lib.qutai_amd_attention_packed_rows(*self.extent, heads, kv_heads, dim, dtype, int(whole),
                                                                     scale, number)
            found = self._plans[key] = (*self.tiles(rows, "length" if not causal else "start" if number == 2 else "end"), rows)
        return found

    def tiles(self, rows, longest_first):
        """(storage, count): for every tile of ``rows`` tokens of a sequence its
        start, its length and the tile's first token in it, as int64 triples (a
        tile per workgroup of attention).  Tiles that have most to do come first:
        causal queries see what lies before them (``longest_first`` "end"), causal
        keys are seen by what lies behind ("start"), and without a mask the work
        goes by the length ("length")."""
        key = rows, longest_first
        if key not in self._tiles:
            tiles = [(n, start, first) for start, n in zip(self.starts, self.lengths) for first in range(0, n, rows)]
            work = {"end": lambda t: -min(t[2] + rows, t[0]), "start": lambda t: t[2] - t[0], "length": lambda t: -t[0]}
            tiles.sort(key=work[longest_first])
            table = array("q", chain.from_iterable((start, n, first) for n, start, first in tiles))
            self._tiles[key] = amd.storage(table, dtype="int64"), len(tiles)
        return self._tiles[key]
