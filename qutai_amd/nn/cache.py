"""Keys and values of earlier positions for causal attention inference
(src/qutai/nn/cache.py:5-29).

The cache holds (batch, heads, length, head_dim) tensors with no graph:
``update`` appends the new positions along the length axis (keys and values
in one launch where their rows are whole 16-byte chunks, else one strided
copy per piece through ``backend.concatenate``) and returns everything
cached so far.

``QuantizedKVCache`` holds the same keys and values in codes of 8 or 4 bits,
quantised as they are written: ``append`` writes new positions in place,
``attend`` is the attention over them, ``read`` gives the values that the
codes stand for.
"""
from __future__ import annotations

from ..backends import amd, amd_lm
from ..backends.device import get_backend
from ..core.tensor import Tensor


def _joined(previous, current):
    if previous is None:
        return Tensor(current.storage.copy(), shape=current.shape)
    batch, heads, length, features = current.shape
    values = get_backend(previous.storage, current.storage).concatenate(
        (previous.storage, current.storage), (previous.shape, current.shape), axis=2)
    return Tensor(values, shape=(batch, heads, previous.shape[2] + length, features))


class KVCache:
    def __init__(self):
        self.keys = None
        self.values = None

    @property
    def length(self) -> int:
        return 0 if self.keys is None else self.keys.shape[2]

    def update(self, keys, values):
        """Append keys and values of shape (batch, heads, new, head_dim);
        returns the cached keys and values of every position."""
        if keys.ndim != 4 or keys.shape != values.shape:
            raise ValueError("cached keys and values need one 4-D shape")
        if self.keys is not None and (self.keys.shape[:2] + self.keys.shape[3:]
                                      != keys.shape[:2] + keys.shape[3:]):
            raise ValueError("new keys and values must match the cache in batch, heads and head size")
        if self.keys is not None and self.keys.shape == self.values.shape:
            batch, heads, past, features = self.keys.shape
            joined = amd_lm.cache_join((self.keys.storage, self.values.storage), (keys.storage, values.storage),
                                       batch * heads)
            if joined is not None:
                shape = (batch, heads, past + keys.shape[2], features)
                self.keys, self.values = (Tensor(x, shape=shape) for x in joined)
                return self.keys, self.values
        self.keys, self.values = _joined(self.keys, keys), _joined(self.values, values)
        return self.keys, self.values


class QuantizedKVCache:
    """Keys and values of up to ``capacity`` positions per sequence, in codes of
    ``bits`` 8 (a scale per head and position) or 4 (a scale per 32 channels of
    it).  Sequences may have different lengths.  Its memory is allocated by the
    first ``append``, which settles batch, heads and head width.  It serves
    inference: what is appended, attended and read has no graph."""

    def __init__(self, capacity, *, bits=8):
        if type(capacity) is not int or capacity <= 0 or bits not in (8, 4):
            raise ValueError("a quantised cache needs a positive capacity and codes of 8 or 4 bits")
        self.capacity, self.bits = capacity, bits
        self.codes = None
        self.lengths = ()
        # lengths[b] is _shift, plus _base[b] where the sequences differ (_stored: _base on the device)
        self._base, self._stored, self._shift = None, None, 0
        self._last = None  # (new, start, starts, counts) of the last append

    @property
    def length(self) -> int:
        """Positions of the longest sequence."""
        return max(self.lengths, default=0)

    def _set_lengths(self, lengths):
        if len(set(lengths)) <= 1:
            self._base, self._stored, self._shift = None, None, lengths[0] if lengths else 0
        elif self._base is not None and all(n - lengths[0] == m - self._base[0] for n, m in zip(lengths, self._base)):
            self._shift = lengths[0] - self._base[0]  # the positions on the device still tell them apart
        else:
            self._base, self._stored, self._shift = lengths, None, 0
        self.lengths = lengths

    def positions(self):
        """(shift, device positions or None) of the next position of every sequence."""
        if self._base is not None and self._stored is None:
            self._stored = amd.storage(self._base, dtype="int64")
        return self._shift, self._stored

    def _per_sequence(self, values, most, what):
        values = (values,) * len(most) if type(values) is int else tuple(values)
        if len(values) != len(most) or any(type(n) is not int or not 0 <= n <= m for n, m in zip(values, most)):
            raise ValueError(f"{what} is one integer per sequence (or one for all), within what there is")
        return values

    def reserve(self, batch, kv_heads, dim):
        """Allocate the cache's memory now, for these sizes."""
        if self.codes is None:
            self.codes = amd_lm.QuantizedCache(batch, kv_heads, dim, self.capacity, self.bits)
            self.lengths = (0,) * batch
        elif (batch, kv_heads, dim) != (self.codes.batch, self.codes.kv_heads, self.codes.dim):
            raise ValueError("new keys and values must match the cache in batch, heads and head size")

    def _state(self):
        """What the cache holds now, for ``_restore``."""
        return self.codes, self.lengths, self._base, self._stored, self._shift, self._last

    def _restore(self, state):
        """Back to an earlier ``_state``, behind which there were appends alone:
        positions truncated in between may have been written again."""
        self.codes, self.lengths, self._base, self._stored, self._shift, self._last = state

    def append(self, keys, values, counts=None):
        """Quantise new positions (batch, new, kv_heads, dim) behind those each
        sequence has; of sequence b only the first ``counts[b]`` where given."""
        if keys.ndim != 4 or keys.shape != values.shape or keys.dtype != values.dtype:
            raise ValueError("cached keys and values need one 4-D shape and one dtype")
        batch, new, kv_heads, dim = keys.shape
        self.append_rows(keys.storage, values.storage, batch, new, kv_heads, dim, counts)

    def append_rows(self, keys, values, batch, new, kv_heads, dim, counts=None, **columns):
        """``append`` of storages, whose positions may be columns of a wider
        matrix (amd_lm.cache_quantize's key_column, key_row, value_column, value_row)."""
        if min(batch, kv_heads, dim) <= 0 or new < 0:
            raise ValueError("cached keys and values need one sequence, head and channel at least")
        counts = (new,) * batch if counts is None else self._per_sequence(counts, (new,) * batch, "counts")
        lengths = tuple(n + m for n, m in zip(self.lengths or (0,) * batch, counts))
        if max(lengths) > self.capacity:
            raise ValueError("the cache's capacity is exceeded")
        first = self.codes is None
        if first:  # (cache_quantize checks them too, but behind reserve)
            amd_lm.cache_rows(keys, values, batch, new, kv_heads, dim, **columns)
        try:
            self.reserve(batch, kv_heads, dim)
            start, starts = self.positions()
            held = None if min(counts) == new else amd.storage(counts, dtype="int64")
            amd_lm.cache_quantize(self.codes, keys, values, new, start=start, starts=starts, counts=held, **columns)
        except BaseException:
            if first:  # a refused call settles nothing
                self.codes, self.lengths = None, ()
            raise
        self._set_lengths(lengths)
        self._last = new, start, starts, held

    def attend(self, queries, *, scale=None):
        """Causal attention of the last ``append``'s positions over everything
        cached: queries (batch, new, heads, dim), heads a multiple of the
        cached ones; the result has their shape and dtype, and is zero at the
        positions that ``counts`` left out.  Nothing is recorded."""
        if self._last is None:
            raise ValueError("attend follows an append: its queries are the positions appended last")
        new, start, starts, counts = self._last
        if queries.ndim != 4 or queries.shape[:2] != (self.codes.batch, new) or queries.shape[3] != self.codes.dim:
            raise ValueError("queries are (batch, new, heads, dim) of the positions appended last")
        out = amd_lm.attention_quantized(self.codes, queries.storage, new, queries.shape[2], start=start, starts=starts,
                                         counts=counts, longest=self.length, scale=scale)
        return Tensor(out, shape=queries.shape)

    def read(self, dtype="float32"):
        """The cached keys and values, (batch, kv_heads, length, dim) each, as
        the codes hold them (rounded to bfloat16 where asked); zeros behind a
        shorter sequence's end."""
        if self.codes is None:
            raise ValueError("nothing was cached yet")
        shift, stored = self.positions()
        c, length = self.codes, self.length
        pair = amd_lm.cache_dequantize(c, length, lengths=stored, shift=shift, dtype=dtype)
        return tuple(Tensor(x, shape=(c.batch, c.kv_heads, length, c.dim)) for x in pair)

    def truncate(self, lengths):
        """Forget the positions from ``lengths`` on (one number for all
        sequences, or one each)."""
        if self.codes is None:
            if any((lengths,) if type(lengths) is int else lengths):
                raise ValueError("nothing was cached yet")
            return
        self._set_lengths(self._per_sequence(lengths, self.lengths, "lengths"))
        self._last = None


class unchanged_on_failure:
    """Context in which quantised caches are appended to: where it raises they
    are as they were before, so that the call may be made again."""

    def __init__(self, *caches):
        self.states = [(cache, cache._state()) for cache in caches]

    def __enter__(self):
        return self

    def __exit__(self, kind, value, traceback):
        if kind is not None:
            for cache, state in self.states:
                cache._restore(state)
