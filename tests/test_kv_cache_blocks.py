"""The cache's book-keeping on the host: blocks given out once, returned, refused
as a whole where there are too few."""

from __future__ import annotations

import numpy as np
import pytest

from mote_amd.kv_cache import BlockTable, CacheFull


def held(t):
    return [int(b) for b in t.table.ravel() if b >= 0]


def test_blocks_are_given_out_once_and_come_back():
    t = BlockTable(8, 3, 128)
    a, b = t.open(), t.open()
    t.reserve([a, b], [33, 1])
    t.advance([a, b], [33, 1])
    assert len(held(t)) == 3 == len(set(held(t))) and t.free_blocks == 5
    t.reserve([b], [31])  # fits the block it has
    t.advance([b], [31])
    assert t.free_blocks == 5
    t.reserve([a], [31])
    assert t.free_blocks == 5
    t.reserve([a], [32])  # reserved, not advanced: the same tokens
    assert t.free_blocks == 4
    t.close(a)
    assert t.free_blocks == 7 and (t.table[a] == -1).all() and t.lengths[a] == 0
    assert t.open() == a


def test_all_or_nothing():
    t = BlockTable(4, 2, 256)
    a, b = t.open(), t.open()
    before = t.table.copy()
    with pytest.raises(CacheFull):
        t.reserve([a, b], [65, 64])
    with pytest.raises(CacheFull):
        t.reserve([a], [257])
    assert np.array_equal(t.table, before) and t.free_blocks == 4
    with pytest.raises(CacheFull):
        t.open()


def test_truncate():
    t = BlockTable(6, 1, 192)
    s = t.open()
    t.reserve([s], [100])
    t.advance([s], [100])
    t.truncate(s, 64)
    assert t.lengths[s] == 64 and t.free_blocks == 4
    t.truncate(s, 33)
    assert t.free_blocks == 4
    t.truncate(s, 0)
    assert t.free_blocks == 6
    with pytest.raises(ValueError):
        t.truncate(s, 1)


def test_refusals():
    t = BlockTable(4, 2, 64)
    s = t.open()
    for call in (lambda: t.reserve([s, s], [1, 1]), lambda: t.reserve([1], [1]), lambda: t.reserve([s], [-1]),
                 lambda: t.close(1), lambda: t.close(-1), lambda: BlockTable(0, 1, 1), lambda: BlockTable(1, 0, 1),
                 lambda: BlockTable(1, 1, 0)):
        with pytest.raises(ValueError):
            call()
