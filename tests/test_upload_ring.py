"""The pinned ring of small uploads: a region is only written again after the copy
that reads it was waited for, and an upload looks at the oldest copies alone
(driver calls are stand-ins: no device)."""
import ctypes
import random
import threading
from array import array
from collections import deque

import pytest

from qutai_amd.backends.amd_runtime import Runtime


class Ring(Runtime):
    STAGING_BYTES = 4096

    def __init__(self):
        self._lock, self._closed = threading.RLock(), False
        self.memory = ctypes.create_string_buffer(self.STAGING_BYTES)
        self._staging, self._staging_at, self._staging_pending = ctypes.addressof(self.memory), 0, deque()
        self.sent, self.waited, self.events, self.large = {}, set(), 0, 0
        self._memcpy = self._large

    def close(self):
        self._closed = True

    def _large(self, *arguments):
        self.large += 1
        return 0

    def _memcpy_async(self, dst, src, nbytes, kind, stream):
        start = src - ctypes.addressof(self.memory)
        for event, (lo, hi) in self.sent.items():
            assert event in self.waited or hi <= start or start + nbytes <= lo
        assert dst == 77 and start + nbytes <= self.STAGING_BYTES and bytes(self.memory[start:start + nbytes]) == self.expected
        self.region = start, start + nbytes
        return 0

    def _event_create_flags(self, out, flags):
        self.events += 1
        out._obj.value = self.events
        return 0

    def _event_record(self, event, stream):
        self.sent[event.value] = self.region
        return 0

    def _event_sync(self, event):
        self.waited.add(event)
        return 0

    def _event_destroy(self, event):
        assert event in self.waited
        del self.sent[event]
        return 0


@pytest.mark.parametrize("seed", range(6))
def test_regions_are_waited_for_before_they_are_written_again(seed):
    rng, ring = random.Random(seed), Ring()
    for _ in range(2000):
        n = rng.choice([1, 8, 256, 257, 700, 1024, rng.randint(1, 1024)])
        data = array("B", rng.randbytes(n))
        ring.expected = data.tobytes()
        ring.upload(77, data)
    assert ring.large == 0 and len(ring.sent) == len(ring._staging_pending) <= 4096 // 256
    ring.upload(77, array("B", bytes(1025)))
    assert ring.large == 1
