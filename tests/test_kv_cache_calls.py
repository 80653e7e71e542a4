"""What KVCacheQ8 uploads and passes on for each call (CPU: stand-in buffers and
entry points that keep what they are given)."""

from __future__ import annotations

import numpy as np
import pytest

from mote_amd import kv_cache

K, V, Q, OUT, STREAM = 0x1000, 0x2000, 0x3000, 0x4000, None


class Buffer:
    """Device memory that holds what was uploaded last."""

    def __init__(self, nbytes):
        self.nbytes, self.ptr = nbytes, id(self)
        self.words = np.full(nbytes // 4, -77, np.int32)

    def upload(self, array):
        flat = np.ascontiguousarray(array).view(np.int32).ravel()
        self.words[: flat.size] = flat


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(kv_cache, "DeviceBuffer", Buffer)
    calls = []
    for name in ("kv_cache_append_q8", "kv_cache_read_q8_f16", "cache_attention_q8_f16"):
        monkeypatch.setattr(kv_cache.ops, name, lambda *a, _name=name, **k: calls.append((_name, a, k)))
    monkeypatch.setattr(kv_cache.ops, "cache_attention_workspace", lambda *a: 0)
    c = kv_cache.KVCacheQ8(12, 2, 64, 4, 128)
    c.calls = calls
    for _ in range(3):
        c.open()
    c.append([0, 1, 2], K, V, [70, 33, 1], STREAM)
    calls.clear()
    return c


def state(cache, n):
    """What the last call finds on the device, and the sizes it was given."""
    name, args, _ = cache.calls[-1]
    return (name, [a for a in args if isinstance(a, int) and a < 1 << 16], cache._offsets.words[: n + 1].tolist(),
            cache._second.words[:n].tolist(), cache._table.words.reshape(-1, cache.blocks.width)[:n].tolist())


FORMS = [tuple, list, np.array, lambda s: np.array(s, np.uint8), lambda s: iter(s)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("sequences", [(0, 1), (2, 0), (1,), (2, 1, 0)])
def test_sequences_in_any_form(cache, sequences, form):
    """A tuple, a list, an array, an iterator: the same tables and lengths."""
    n = len(sequences)
    table = [cache.blocks.table[s].tolist() for s in sequences]
    lengths = [cache.length(s) for s in sequences]
    cache.read(form(sequences), K, V, form([1] * n), form([0] * n), STREAM)
    assert state(cache, n)[0] == "kv_cache_read_q8_f16"
    assert state(cache, n)[2:] == (list(range(n + 1)), [0] * n, table)
    cache.attend(form(sequences), Q, OUT, 4, form([1] * n), STREAM)
    assert state(cache, n)[0] == "cache_attention_q8_f16"
    assert state(cache, n)[2:] == (list(range(n + 1)), lengths, table)
    cache.append(form(sequences), K, V, form([2] * n), STREAM)
    assert state(cache, n)[0] == "kv_cache_append_q8"
    assert state(cache, n)[2:] == (list(range(0, 2 * n + 1, 2)), lengths, [cache.blocks.table[s].tolist() for s in sequences])
    assert [cache.length(s) for s in sequences] == [t + 2 for t in lengths]


def test_no_sequence(cache):
    for none in ((), [], np.array([], np.int64)):
        cache.append(none, K, V, none, STREAM)
        cache.read(none, K, V, none, none, STREAM)
        cache.attend(none, Q, OUT, 4, none, STREAM)
    assert cache.blocks.lengths.tolist() == [70, 33, 1, 0]


def test_refused_calls_leave_the_cache_as_it_was(cache):
    free, table = cache.blocks.free_blocks, cache.blocks.table.copy()
    for sequences in ((0, 0), (0, 3), (-1,), (0.0, 1.0), ("0",)):
        n = len(sequences)
        with pytest.raises((ValueError, TypeError)):
            cache.append(sequences, K, V, [40] * n, STREAM)
        with pytest.raises((ValueError, TypeError)):
            cache.read(sequences, K, V, [1] * n, [0] * n, STREAM)
        with pytest.raises((ValueError, TypeError)):
            cache.attend(sequences, Q, OUT, 4, [1] * n, STREAM)
    for counts in ((1,), (1, 1, 1), (1, 0.5)):
        with pytest.raises((ValueError, TypeError)):
            cache.append((0, 1), K, V, counts, STREAM)
    assert not cache.calls and cache.blocks.free_blocks == free
    assert np.array_equal(cache.blocks.table, table) and cache.blocks.lengths.tolist() == [70, 33, 1, 0]
