"""Scores as large as finite binary16 queries and keys can make them: outputs stay
finite and right.  Equal keys weigh the same whatever their score, and a key whose
score is far above the others' takes all the weight."""

from __future__ import annotations

import numpy as np
import pytest

from attention_oracle import BLOCK, Cache, assert_within
from mote_amd import ops
from mote_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu

# Of queries and keys: scores in powers of two from 2^19 to 2^37 for heads of 64.
SIZES = [2.0**e * f for e in range(8, 16) for f in (1.0, 1.25, 1.5, 1.75)]


def mean_within(v, seen):
    """Means of v over the keys each row sees, and what equal weights may be off by:
    each is rounded to f16 once (2^-11) where its sum is not, sums over t keys are in
    f32 (t 2^-23), the output is rounded to f16 (2^-11, 2^-25 where subnormal)."""
    w = seen / seen.sum(1, keepdims=True)
    t = v.shape[0]
    o = np.einsum("nt,thd->nhd", w, v)
    size = np.einsum("nt,thd->nhd", w, np.abs(v))
    return o, 2.0**-11 * np.abs(o) + size * (2.0**-11 + (t + 2) * 2.0**-23) + 2.0**-24


def one_within(v, at):
    o = v[at]
    return o, np.abs(o) * (2.0**-11 + 2.0**-11 + 4 * 2.0**-23) + 2.0**-24


def queries_of(n, heads, d):
    """Row i's entries: all SIZES in turn, over rows and heads."""
    i = np.arange(n * heads).reshape(n, heads, 1)
    return np.broadcast_to(np.array(SIZES)[i % len(SIZES)], (n, heads, d)).astype(np.float16)


def rows_seen(n, t):
    return (np.arange(t)[None, :] <= np.arange(n)[:, None] + t - n).astype(np.float64)


def prompt(stream, q, k, v):
    n, heads, d = q.shape
    t, kv_heads = k.shape[:2]
    bufs = [DeviceBuffer.from_array(x) for x in (q, k, v)]
    at = [DeviceBuffer.from_array(np.array(x, np.int32)) for x in ([0, n], [0, t])]
    sizes = (1, n, t, t, heads, kv_heads, d)
    need = ops.prompt_attention_workspace(*sizes)
    out, work = DeviceBuffer(q.nbytes), DeviceBuffer(need)
    ops.prompt_attention_f16(*(b.ptr for b in bufs), out.ptr, *(b.ptr for b in at), *sizes, d ** -0.5, work.ptr, need,
                             stream)
    stream.synchronize()
    return out.download(np.float16).reshape(q.shape)


PROMPTS = [(100, 100, 64, 4, 2), (33, 200, 40, 2, 1), (70, 70, 128, 128, 4), (5, 3000, 128, 4, 2), (9, 150, 256, 2, 2)]


@pytest.mark.parametrize("n,t,d,heads,kv_heads", PROMPTS)
@pytest.mark.parametrize("key", [200.0, 1000.0, 3000.0, -3000.0, 65504.0])
def test_prompts_equal_keys(stream, n, t, d, heads, kv_heads, key):
    rng = np.random.default_rng(1)
    q = queries_of(n, heads, d)
    k = np.full((t, kv_heads, d), key, np.float16)
    v = rng.standard_normal((t, kv_heads, d)).astype(np.float16)
    o, bound = mean_within(v.astype(np.float64), rows_seen(n, t))
    group = heads // kv_heads
    assert_within(prompt(stream, q, k, v), o.repeat(group, 1), bound.repeat(group, 1))


@pytest.mark.parametrize("n,t,d,heads,kv_heads", PROMPTS)
@pytest.mark.parametrize("key", [1000.0, 65504.0])
def test_prompts_one_key_above_the_others(stream, n, t, d, heads, kv_heads, key):
    """The first, one that all rows see in the middle, and each row's own."""
    rng = np.random.default_rng(2)
    v = rng.standard_normal((t, kv_heads, d)).astype(np.float16)
    group = heads // kv_heads
    for at in (0, (t - n) // 2):
        k = np.full((t, kv_heads, d), -key, np.float16)
        k[at] = key
        o, bound = one_within(v.astype(np.float64), np.full(n, at))
        assert_within(prompt(stream, queries_of(n, heads, d), k, v), o.repeat(group, 1), bound.repeat(group, 1))
    # growing keys: steps of 1/64 of the key, past any rounding of the score
    steps = np.minimum(np.arange(t) * 64 // t, 63)
    k = (key * (steps + 1) / 64)[:, None, None] * np.ones((1, kv_heads, d))
    first = np.searchsorted(steps, steps)
    seen = rows_seen(n, t)
    rows = np.arange(n) + t - n
    same = (np.arange(t)[None, :] >= first[rows][:, None]) * seen
    o, bound = mean_within(v.astype(np.float64), same)
    assert_within(prompt(stream, queries_of(n, heads, d), k.astype(np.float16), v), o.repeat(group, 1),
                  bound.repeat(group, 1))


CACHES = [(1, 300, 128, 8, 2), (3, 100, 64, 4, 2), (3, 3000, 64, 4, 2), (20, 300, 64, 4, 2), (3, 300, 256, 4, 2),
          (60, 500, 64, 4, 2), (60, 3000, 64, 4, 2), (40, 300, 256, 4, 2)]


@pytest.mark.parametrize("n,t,d,heads,kv_heads", CACHES)
@pytest.mark.parametrize("key", [200.0, 1000.0, 3000.0, -3000.0, 65504.0])
def test_cache_equal_keys(stream, n, t, d, heads, kv_heads, key):
    """All blocks' scales are the same; those of keys make 100 the key's size."""
    rng = np.random.default_rng(3)
    blocks = -(-t // BLOCK)
    host = Cache(blocks, kv_heads, d, rng)
    host.bytes[:, :, 0] = 128 + int(np.copysign(100, key))
    host.scales[:, :, 0], host.scales[:, :, 1] = abs(key) / 100, 0.0125
    table = rng.permutation(blocks).astype(np.int32)
    q = queries_of(n, heads, d)
    bufs = [DeviceBuffer.from_array(x) for x in (q, host.bytes, host.scales)]
    lists = [DeviceBuffer.from_array(np.array(x, np.int32)) for x in ([0, n], [t], table)]
    sizes = (1, n, n, t, heads, kv_heads, d)
    need = ops.cache_attention_workspace(*sizes)
    out, work = DeviceBuffer(q.nbytes), DeviceBuffer(need)
    ops.cache_attention_q8_f16(*(b.ptr for b in bufs), *(b.ptr for b in lists), out.ptr, *sizes, blocks, blocks,
                               d ** -0.5, work.ptr, need, stream)
    stream.synchronize()
    o, bound = mean_within(host.values(1, table, t).astype(np.float64), rows_seen(n, t))
    group = heads // kv_heads
    assert_within(out.download(np.float16).reshape(q.shape), o.repeat(group, 1), bound.repeat(group, 1))
