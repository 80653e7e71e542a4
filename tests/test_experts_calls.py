"""What ExpertsMX refuses before it takes any memory, and the streams it waits for
(CPU: stand-in buffers and entry points)."""

from __future__ import annotations

import numpy as np
import pytest

from mote_amd import experts, ops


class Buffer:
    taken = 0

    def __init__(self, nbytes):
        Buffer.taken += 1
        self.nbytes, self.ptr = nbytes, 0x1000

    @classmethod
    def from_array(cls, array):
        return cls(array.nbytes)


@pytest.fixture
def buffers(monkeypatch):
    monkeypatch.setattr(experts, "DeviceBuffer", Buffer)
    Buffer.taken = 0
    return Buffer


GOOD = dict(experts=16, top=4, hidden=64, inner=96, max_tokens=5, groups=4, top_groups=2)
REFUSED = [dict(experts=0), dict(experts=1025, groups=1, top_groups=1), dict(top=0), dict(top=17),
           dict(experts=128, top=65, groups=1, top_groups=1), dict(top=9), dict(hidden=33), dict(hidden=0),
           dict(inner=1 << 25), dict(max_tokens=0), dict(max_tokens=1 << 29), dict(bits=8), dict(score=2), dict(score=-1),
           dict(groups=0), dict(groups=3), dict(top_groups=0), dict(top_groups=5), dict(group_best=0), dict(group_best=3),
           dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e39), dict(bias=np.zeros(15))]


def test_what_is_allowed(buffers):
    layer = experts.ExpertsMX(**GOOD)
    assert buffers.taken > 0 and layer.top == 4
    experts.ExpertsMX(1024, 64, 64, 96, 5)


@pytest.mark.parametrize("change", REFUSED, ids=str)
def test_refusals_before_any_memory(buffers, change):
    with pytest.raises(ValueError):
        experts.ExpertsMX(**{**GOOD, **change})
    assert buffers.taken == 0


@pytest.mark.parametrize("by_handle", [False, True])
def test_load_waits_for_a_stream_or_its_handle(buffers, monkeypatch, by_handle):
    events = []
    monkeypatch.setattr(experts.ops, "mx_quantize_f32", lambda *a: events.append(("quantize", ops._s(a[-1]))))

    class Library:
        @staticmethod
        def mote_hip_stream_synchronize(handle):
            events.append(("wait", handle))
            return 0

    monkeypatch.setattr(experts, "lib", Library, raising=False)

    class Stream:
        handle = 0x77

        def synchronize(self):
            events.append(("wait", self.handle))

    layer = experts.ExpertsMX(**GOOD)
    gate = np.zeros((96, 64), np.float32)
    layer.load(3, gate, gate, np.zeros((64, 96), np.float32), Stream.handle if by_handle else Stream())
    assert events == [("quantize", 0x77)] * 3 + [("wait", 0x77)]
