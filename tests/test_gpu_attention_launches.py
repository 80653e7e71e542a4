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
