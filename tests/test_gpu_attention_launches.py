"""Calls of more workgroups than one launch has room for."""

from __future__ import annotations

import numpy as np
import pytest

from attention_oracle import BLOCK, Cache, assert_within, attend
from mote_amd import ops
from mote_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu

SENTINEL = 0x7A7A


def test_cache_attention_of_half_a_million_sequences(stream):
    """One token each over one block, eight key heads: 4 194 344 workgroups of 1024
    threads, and a launch has room for 4 194 303.  Blocks are shared for reading."""
    rng = np.random.default_rng(1)
    sequences, heads, d = 524293, 8, 8
    host = Cache(16, heads, d, rng)
    q = rng.standard_normal((sequences, heads, d), dtype=np.float32).astype(np.float16)
    lengths = rng.integers(0, BLOCK + 1, sequences).astype(np.int32)
    table = rng.integers(0, 16, (sequences, 1)).astype(np.int32)
    bufs = [DeviceBuffer.from_array(x) for x in (q, host.bytes, host.scales)]
    lists = [DeviceBuffer.from_array(x) for x in (lengths, table)]
    out = DeviceBuffer.from_array(np.full(q.size, SENTINEL, np.uint16))
    sizes = (sequences, sequences, 1, BLOCK, heads, heads, d)
    assert ops.cache_attention_workspace(*sizes) == 0
    ops.cache_attention_q8_f16(*(b.ptr for b in bufs), None, *(b.ptr for b in lists), out.ptr, *sizes, 1, 16,
                               d ** -0.5, 0, 0, stream)
    stream.synchronize()
    got = out.download(np.float16).reshape(q.shape)
    assert (got.view(np.uint16) != SENTINEL).all()
    assert (got[lengths == 0] == 0).all()
    for s in [*range(200), *range(sequences - 200, sequences), *rng.integers(0, sequences, 200).tolist()]:
        k, v = (host.values(w, table[s], lengths[s]).astype(np.float64) for w in (0, 1))
        o, bound = attend(q[s:s + 1], k, v, d ** -0.5)
        assert_within(got[s:s + 1], o, bound, f"sequence {s}")


def test_cache_writes_and_reads_of_eight_million_sequences(stream):
    """One token each: more than the 16 777 215 workgroups of 256 threads a launch has
    room for.  Blocks for the first, the last and some between; the others have none."""
    rng = np.random.default_rng(2)
    sequences, heads, d = (1 << 23) + 9, 1, 8
    held = np.unique(np.concatenate([np.arange(20), sequences - 1 - np.arange(20), rng.integers(0, sequences, 60)]))
    host = Cache(len(held), heads, d, rng)
    table = np.full((sequences, 1), -1, np.int32)
    table[held, 0] = rng.permutation(len(held))
    positions = rng.integers(0, BLOCK, sequences).astype(np.int32)
    k, v = (rng.standard_normal((sequences, heads, d), dtype=np.float32).astype(np.float16) for _ in range(2))
    kb, vb, at, pos, tab, cache, scales = (DeviceBuffer.from_array(x) for x in (
        k, v, np.arange(sequences + 1, dtype=np.int32), positions, table, host.bytes, host.scales))
    ops.kv_cache_append_q8(kb.ptr, vb.ptr, at.ptr, pos.ptr, tab.ptr, cache.ptr, scales.ptr, sequences, sequences, heads,
                           d, 1, len(held), stream)
    back = [DeviceBuffer.from_array(np.full(k.size, SENTINEL, np.uint16)) for _ in range(2)]
    ops.kv_cache_read_q8_f16(cache.ptr, scales.ptr, at.ptr, pos.ptr, tab.ptr, back[0].ptr, back[1].ptr, sequences,
                             sequences, heads, d, 1, len(held), stream)
    stream.synchronize()
    for s in held:
        for which, x in ((0, k), (1, v)):
            host.append(x[s:s + 1], which, table[s], positions[s])
    assert (cache.download(np.uint8).reshape(host.bytes.shape) == host.bytes).all()
    assert (scales.download(np.float32).reshape(host.scales.shape) == host.scales).all()
    for which in (0, 1):
        got = back[which].download(np.uint16).reshape(k.shape)
        for s in held:
            want = host.values(which, table[s], positions[s] + 1)[-1:].astype(np.float16)
            assert (got[s:s + 1] == want.view(np.uint16)).all()
        got[held] = SENTINEL
        assert (got == SENTINEL).all()


def test_prompts_of_many_sequences_and_heads(stream):
    """70000 sequences of one token, whose attention is its value, with 512 heads: more
    than 2^32 threads in a launch's three directions together."""
    rng = np.random.default_rng(3)
    sequences, heads, d = 70000, 512, 8
    v = rng.integers(0, 0x7C00, (sequences, heads, d), dtype=np.uint16)
    q = rng.integers(0, 0x4000, v.shape, dtype=np.uint16)
    qb, vb = DeviceBuffer.from_array(q), DeviceBuffer.from_array(v)
    at = DeviceBuffer.from_array(np.arange(sequences + 1, dtype=np.int32))
    out = DeviceBuffer(v.nbytes)
    sizes = (sequences, sequences, sequences, 1, heads, heads, d)
    assert ops.prompt_attention_workspace(*sizes) == 0
    ops.prompt_attention_f16(qb.ptr, qb.ptr, vb.ptr, out.ptr, at.ptr, None, *sizes, d ** -0.5, 0, 0, stream)
    stream.synchronize()
    assert (out.download(np.uint16).reshape(v.shape) == v).all()


def test_cache_writes_and_reads_of_many_sequences_and_heads(stream):
    """As many workgroups, in two directions: 2^18 sequences of one token, 128 heads.
    One sequence in 4096 has a block."""
    rng = np.random.default_rng(4)
    sequences, heads, d = 1 << 18, 128, 8
    held = np.arange(4095, sequences, 4096)
    host = Cache(len(held), heads, d, rng)
    table = np.full((sequences, 1), -1, np.int32)
    table[held, 0] = rng.permutation(len(held))
    positions = rng.integers(0, BLOCK, sequences).astype(np.int32)
    k, v = (rng.integers(0, 0x4000, (sequences, heads, d), dtype=np.uint16).view(np.float16) for _ in range(2))
    kb, vb, at, pos, tab, cache, scales = (DeviceBuffer.from_array(x) for x in (
        k, v, np.arange(sequences + 1, dtype=np.int32), positions, table, host.bytes, host.scales))
    ops.kv_cache_append_q8(kb.ptr, vb.ptr, at.ptr, pos.ptr, tab.ptr, cache.ptr, scales.ptr, sequences, sequences, heads,
                           d, 1, len(held), stream)
    back = [DeviceBuffer.from_array(np.full(k.size, SENTINEL, np.uint16)) for _ in range(2)]
    ops.kv_cache_read_q8_f16(cache.ptr, scales.ptr, at.ptr, pos.ptr, tab.ptr, back[0].ptr, back[1].ptr, sequences,
                             sequences, heads, d, 1, len(held), stream)
    stream.synchronize()
    for s in held:
        for which, x in ((0, k), (1, v)):
            host.append(x[s:s + 1], which, table[s], positions[s])
    assert (cache.download(np.uint8).reshape(host.bytes.shape) == host.bytes).all()
    for which in (0, 1):
        got = back[which].download(np.uint16).reshape(k.shape)
        for s in held:
            want = host.values(which, table[s], positions[s] + 1)[-1:].astype(np.float16)
            assert (got[s:s + 1] == want.view(np.uint16)).all()
        got[held] = SENTINEL
        assert (got == SENTINEL).all()
