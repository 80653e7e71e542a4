"""The cache's class, and the example that runs the attention block from prompts
to generated tokens."""

from __future__ import annotations

import importlib.util
import os

import numpy as np
import pytest

from attention_oracle import Cache, assert_within, attend
from mote_amd.device import DeviceBuffer, Stream
from mote_amd.kv_cache import CacheFull, KVCacheQ8

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rows(rng, n, heads, d):
    return rng.standard_normal((n, heads, d)).astype(np.float16)


def test_cache_class(stream):
    """Sequences that start, go on, go back and end; every step's attention and
    what is read back against the host's cache."""
    rng = np.random.default_rng(1)
    kv_heads, heads, d = 2, 6, 64
    cache = KVCacheQ8(12, kv_heads, d, 3, 160)
    tokens = {}

    def append(sequences, counts):
        k, v = (rows(rng, sum(counts), kv_heads, d) for _ in range(2))
        kb, vb = DeviceBuffer.from_array(k), DeviceBuffer.from_array(v)
        before = [cache.length(s) for s in sequences]
        cache.append(sequences, kb.ptr, vb.ptr, counts, stream)
        stream.synchronize()
        at = 0
        for s, n, p in zip(sequences, counts, before):
            host = tokens[s]
            host.append(k[at:at + n], 0, list(range(5)), p)
            host.append(v[at:at + n], 1, list(range(5)), p)
            at += n

    def attend_all(sequences, counts, window=0):
        q = rows(rng, sum(counts), heads, d)
        qb, out = DeviceBuffer.from_array(q), DeviceBuffer(q.nbytes)
        cache.attend(sequences, qb.ptr, out.ptr, heads, counts, stream, window=window)
        stream.synchronize()
        got = out.download(np.float16).reshape(q.shape)
        at = 0
        for s, n in zip(sequences, counts):
            k, v = (tokens[s].values(w, list(range(5)), cache.length(s)).astype(np.float64) for w in (0, 1))
            o, bound = attend(q[at:at + n], k, v, d ** -0.5, True, window)
            assert_within(got[at:at + n], o, bound)
            at += n

    a, b = cache.open(), cache.open()
    tokens[a], tokens[b] = Cache(5, kv_heads, d), Cache(5, kv_heads, d)
    append([a, b], [50, 3])
    attend_all([a, b], [50, 3])
    for _ in range(35):
        append([b, a], [1, 1])
    attend_all([a], [1])
    attend_all([b, a], [1, 2], window=20)
    cache.truncate(a, 70)
    append([a], [5])
    attend_all([a, b], [5, 1])
    k = DeviceBuffer(2 * 40 * kv_heads * d)
    v = DeviceBuffer(k.nbytes)
    cache.read([a], k.ptr, v.ptr, [40], [30], stream)
    stream.synchronize()
    want = tokens[a].values(0, list(range(5)), 70)[30:].astype(np.float16)
    assert (k.download(np.uint16).reshape(want.shape) == want.view(np.uint16)).all()
    with pytest.raises(CacheFull):
        cache.append([a], k.ptr, v.ptr, [160], stream)
    with pytest.raises(ValueError):
        cache.read([a], k.ptr, v.ptr, [40], [40], stream)
    with pytest.raises(ValueError):
        cache.attend([b], k.ptr, v.ptr, heads, [1000], stream)
    cache.close(a)
    other = Stream()  # calls on different streams, one of them gone since
    for s in (other, stream, other, stream):
        qb = DeviceBuffer.from_array(rows(rng, 1, heads, d))
        out = DeviceBuffer(qb.nbytes)
        cache.attend([b], qb.ptr, out.ptr, heads, [1], s)
        if s is other:
            first = out
    other.close()
    attend_all([b], [1])
    assert np.isfinite(first.download(np.float16)).all()
    with pytest.raises(ValueError):
        cache.attend([a], k.ptr, v.ptr, heads, [1], stream)
    cache.free()


@pytest.mark.parametrize("sizes", [dict(hidden=256, heads=4, kv_heads=2, head_dim=64, prompts=(40, 1, 130), steps=5),
                                   dict(hidden=512, heads=4, kv_heads=4, head_dim=128, prompts=(33,), steps=3)])
def test_example(sizes):
    """Keys and values in 8 bits: an element is off by half a step at most, 1/254 of
    its block's largest, about 4 times its root mean square: 1.6 % of it, a third of
    that on average in size (uniform rounding: 0.9 %).  Scores of unit queries and
    keys are then off by 0.9 % of one, weights by as much, and outputs by that and
    the values' 0.9 % at most, with no token averaged away: 2 % of the output's
    size is one standard deviation, six of them the largest of its elements."""
    spec = importlib.util.spec_from_file_location("decoder_attention",
                                                  os.path.join(ROOT, "examples", "decoder_attention.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.run(**sizes) < 0.12
