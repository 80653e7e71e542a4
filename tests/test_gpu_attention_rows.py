"""Which output rows attention writes: those of the sequences' queries, up to
`max_queries` of each over the cache, whether or not the keys are divided into
parts; every other row keeps what it held, whatever the workspace held."""

from __future__ import annotations

import numpy as np
import pytest

from attention_oracle import BLOCK, Cache, assert_within, attend
from mote_amd import ops
from mote_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu

SENTINEL = 0x7A7A
# Workspaces hold numbers that a join would take for statistics and sums: 1.0.
ONES = 0x3F800000


def ints(x):
    return np.asarray(x, np.int32)


def outputs(rows, heads, d):
    return DeviceBuffer.from_array(np.full(rows * heads * d, SENTINEL, np.uint16))


def workspace(need):
    return DeviceBuffer.from_array(np.full(max(need, 4) // 4, ONES, np.uint32))


def check_rows(got, want, bound, computed):
    assert_within(got[computed], want[computed], bound[computed])
    assert (got.view(np.uint16)[~computed] == SENTINEL).all()


def cache_case(stream, seed, at, tokens, lengths, max_queries, heads, kv_heads, d, in_parts):
    """at: the query offsets; tokens: the rows there are."""
    rng = np.random.default_rng(seed)
    blocks = -(-max(lengths) // BLOCK)
    host = Cache(len(lengths) * blocks, kv_heads, d, rng)
    table = rng.permutation(len(host.bytes)).reshape(len(lengths), blocks).astype(np.int32)
    q = rng.standard_normal((tokens, heads, d)).astype(np.float16)
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    computed = np.zeros(tokens, bool)
    for s, t in enumerate(lengths):
        a, n = at[s], at[s + 1] - at[s]
        if n == 0:
            continue
        k, v = (host.values(w, table[s], t).astype(np.float64) for w in (0, 1))
        want[a:a + n], bound[a:a + n] = attend(q[a:a + n], k, v, d ** -0.5)
        computed[a:a + min(n, max_queries)] = True
    bufs = [DeviceBuffer.from_array(x) for x in (q, host.bytes, host.scales, ints(at), ints(lengths), table)]
    sizes = (len(lengths), tokens, max_queries, max(lengths), heads, kv_heads, d)
    need = ops.cache_attention_workspace(*sizes)
    assert (need > 0) == in_parts
    out, work = outputs(tokens, heads, d), workspace(need)
    ops.cache_attention_q8_f16(*(b.ptr for b in bufs), out.ptr, *sizes, blocks, len(host.bytes), d ** -0.5, work.ptr,
                               need, stream)
    stream.synchronize()
    check_rows(out.download(np.float16).reshape(q.shape), want, bound, computed)


CACHE_FORMS = [  # heads, key heads, head size, most queries, lengths, in parts
    (4, 2, 64, 3, [300, 70], False),        # 16-row tiles
    (4, 2, 64, 3, [3000, 700], True),
    (4, 2, 256, 3, [3000, 700], True),
    (4, 2, 64, 20, [300, 70], False),       # 32-row tiles
    (4, 2, 64, 20, [3000, 700], True),
    (4, 2, 64, 60, [300, 70], False),       # 128-row tiles
    (4, 2, 64, 60, [3000, 700], True),
    (4, 2, 256, 60, [3000, 700], True),
]


@pytest.mark.parametrize("heads,kv_heads,d,most,lengths,parts", CACHE_FORMS)
def test_cache_rows_past_the_last_offset(stream, heads, kv_heads, d, most, lengths, parts):
    """A padded batch: rows that belong to no sequence, at the end and at the start."""
    n = most - 1
    cache_case(stream, 1, [0, n, n + most], n + most + 5, lengths, most, heads, kv_heads, d, parts)
    cache_case(stream, 2, [3, 3 + n, 3 + n + most], n + most + 3, lengths, most, heads, kv_heads, d, parts)


@pytest.mark.parametrize("heads,kv_heads,d,most,lengths,parts", CACHE_FORMS)
def test_cache_rows_past_the_stated_most(stream, heads, kv_heads, d, most, lengths, parts):
    """A sequence with more queries than max_queries: its first are computed, at
    the positions that all of them give."""
    cache_case(stream, 3, [0, most + 2, 2 * most + 1], 2 * most + 1, lengths, most, heads, kv_heads, d, parts)
    cache_case(stream, 4, [0, most, 2 * most + 40], 2 * most + 41, lengths, most, heads, kv_heads, d, parts)


def test_cache_rows_of_many_sequences(stream):
    """More than a wave looks up at once, some without a query, some with too many."""
    rng = np.random.default_rng(5)
    lengths = rng.integers(20, 1200, 150).tolist()
    lengths[77] = 3000
    at = np.concatenate([[0], np.cumsum(rng.choice([0, 0, 1, 2, 5], 150))])
    cache_case(stream, 5, at.tolist(), int(at[-1]) + 4, lengths, 2, 2, 1, 32, True)


@pytest.mark.parametrize("keys,in_parts", [([90, 40], False), ([4000, 900], True)])
@pytest.mark.parametrize("d", [40, 128])
@pytest.mark.parametrize("start", [0, 6])
def test_prompt_rows_past_the_last_offset(stream, keys, in_parts, d, start):
    rng = np.random.default_rng(6)
    queries, heads, kv_heads = [9, 4], 4, 2
    tokens = start + sum(queries) + 7
    at = ints([start, start + 9, start + 13])
    q = rng.standard_normal((tokens, heads, d)).astype(np.float16)
    k, v = (rng.standard_normal((sum(keys), kv_heads, d)).astype(np.float16) for _ in range(2))
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    computed = np.zeros(tokens, bool)
    j = 0
    for s, t in enumerate(keys):
        rows = slice(at[s], at[s + 1])
        want[rows], bound[rows] = attend(q[rows], k[j:j + t], v[j:j + t], d ** -0.5)
        computed[rows] = True
        j += t
    bufs = [DeviceBuffer.from_array(x) for x in (q, k, v)]
    offsets = [DeviceBuffer.from_array(x) for x in (at, ints([0, keys[0], sum(keys)]))]
    sizes = (2, tokens, sum(keys), max(keys), heads, kv_heads, d)
    need = ops.prompt_attention_workspace(*sizes)
    assert (need > 0) == in_parts
    out, work = outputs(tokens, heads, d), workspace(need)
    ops.prompt_attention_f16(*(b.ptr for b in bufs), out.ptr, *(b.ptr for b in offsets), *sizes, d ** -0.5, work.ptr,
                             need, stream)
    stream.synchronize()
    check_rows(out.download(np.float16).reshape(q.shape), want, bound, computed)


@pytest.mark.parametrize("heads,kv_heads,d,most,lengths,parts", CACHE_FORMS)
def test_cache_output_over_the_queries(stream, heads, kv_heads, d, most, lengths, parts):
    rng = np.random.default_rng(7)
    blocks = -(-max(lengths) // BLOCK)
    host = Cache(2 * blocks, kv_heads, d, rng)
    table = rng.permutation(2 * blocks).reshape(2, blocks).astype(np.int32)
    q = rng.standard_normal((2 * most - 1, heads, d)).astype(np.float16)
    qb, *bufs = (DeviceBuffer.from_array(x) for x in (q, host.bytes, host.scales, ints([0, most - 1, 2 * most - 1]),
                                                      ints(lengths), table))
    sizes = (2, len(q), most, max(lengths), heads, kv_heads, d)
    need = ops.cache_attention_workspace(*sizes)
    assert (need > 0) == parts
    out, work = outputs(len(q), heads, d), workspace(need)
    for to in (out, qb):
        ops.cache_attention_q8_f16(qb.ptr, *(b.ptr for b in bufs), to.ptr, *sizes, blocks, len(host.bytes), d ** -0.5,
                                   work.ptr, need, stream)
    stream.synchronize()
    assert (qb.download(np.uint16) == out.download(np.uint16)).all()


@pytest.mark.parametrize("d", [40, 128, 256])
def test_prompt_output_over_the_queries_in_parts(stream, d):
    rng = np.random.default_rng(8)
    q = rng.standard_normal((130, 4, d)).astype(np.float16)
    k, v = (rng.standard_normal((3000, 2, d)).astype(np.float16) for _ in range(2))
    qb, kb, vb, at, key_at = (DeviceBuffer.from_array(x) for x in (q, k, v, ints([0, 130]), ints([0, 3000])))
    sizes = (1, 130, 3000, 3000, 4, 2, d)
    need = ops.prompt_attention_workspace(*sizes)
    assert need > 0
    out, work = outputs(130, 4, d), workspace(need)
    for to in (out, qb):
        ops.prompt_attention_f16(qb.ptr, kb.ptr, vb.ptr, to.ptr, at.ptr, key_at.ptr, *sizes, d ** -0.5, work.ptr, need,
                                 stream)
    stream.synchronize()
    assert (qb.download(np.uint16) == out.download(np.uint16)).all()
