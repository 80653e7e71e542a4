"""Every form of the attentions on what the other tests ask of the small ones: the
cache's 128-row tiles with windows, missing blocks, scales that are not numbers,
a context past the stated most and keys in parts; prompts whose keys are in parts
with values that are not finite; and each single key's weight, so that none can be
lost or counted twice between tiles and parts."""

from __future__ import annotations

import numpy as np
import pytest

from attention_oracle import BLOCK, Cache, assert_within, attend
from mote_amd import ops
from mote_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu


def offsets(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def cache_attention(stream, host, table, q, queries, lengths, window=0, max_context=None):
    """(output, whether the keys were in parts)"""
    bufs = [DeviceBuffer.from_array(x) for x in (q, host.bytes, host.scales)]
    lists = [DeviceBuffer.from_array(x) for x in (offsets(queries), np.array(lengths, np.int32),
                                                  np.ascontiguousarray(table, np.int32))]
    heads, d = q.shape[1:]
    sizes = (len(queries), len(q), max(queries), max_context or max(lengths), heads, host.heads, d)
    need = ops.cache_attention_workspace(*sizes)
    out, work = DeviceBuffer(q.nbytes), DeviceBuffer(need)
    ops.cache_attention_q8_f16(*(b.ptr for b in bufs), *(b.ptr for b in lists), out.ptr, *sizes, table.shape[1],
                               len(host.bytes), d ** -0.5, work.ptr, need, stream, window=window)
    stream.synchronize()
    return out.download(np.float16).reshape(q.shape), need > 0


def prompt_attention(stream, q, k, v, queries, keys, window=0):
    bufs = [DeviceBuffer.from_array(x) for x in (q, k, v)]
    lists = [DeviceBuffer.from_array(offsets(x)) for x in (queries, keys)]
    heads, d = q.shape[1:]
    sizes = (len(queries), len(q), len(k), max(keys), heads, k.shape[1], d)
    need = ops.prompt_attention_workspace(*sizes)
    out, work = DeviceBuffer(q.nbytes), DeviceBuffer(need)
    ops.prompt_attention_f16(*(b.ptr for b in bufs), out.ptr, *(b.ptr for b in lists), *sizes, d ** -0.5, work.ptr,
                             need, stream, window=window)
    stream.synchronize()
    return out.download(np.float16).reshape(q.shape), need > 0


def setup(seed, queries, lengths, heads, kv_heads, d):
    rng = np.random.default_rng(seed)
    blocks = -(-max(lengths) // BLOCK)
    host = Cache(len(lengths) * blocks + 2, kv_heads, d, rng)
    table = rng.permutation(len(host.bytes))[: len(lengths) * blocks].reshape(len(lengths), blocks).astype(np.int32)
    return host, table, (1.5 * rng.standard_normal((sum(queries), heads, d))).astype(np.float16)


def expected(host, table, q, queries, lengths, window=0):
    o, b = np.zeros(q.shape), np.zeros(q.shape)
    row = 0
    for s, (n, t) in enumerate(zip(queries, lengths)):
        k, v = (host.values(w, table[s], t).astype(np.float64) for w in (0, 1))
        o[row:row + n], b[row:row + n] = attend(q[row:row + n], k, v, q.shape[2] ** -0.5, True, window)
        row += n
    return o, b


# Rows of a key head (queries x 2) that take 128-row tiles: more than 96 for heads of
# up to 128 dimensions, more than 64 above.
TILES = [(60, 32), (60, 64), (70, 96), (60, 128), (40, 160), (40, 256)]


@pytest.mark.parametrize("n,d", TILES)
@pytest.mark.parametrize("window", [1, 33, 64, 299, 1 << 40])
@pytest.mark.parametrize("lengths,parts", [([300, 77, 30], False), ([2600, 700, 1], True)])
def test_cache_tiles_windows(stream, n, d, window, lengths, parts):
    queries = [n, n, 5]
    host, table, q = setup(d, queries, lengths, 4, 2, d)
    got, in_parts = cache_attention(stream, host, table, q, queries, lengths, window)
    assert in_parts or not parts
    assert_within(got, *expected(host, table, q, queries, lengths, window))


def attend_at(q, k, v, positions, keys):
    """Queries at `positions` over the tokens `keys` alone."""
    o, bound = np.zeros(q.shape), np.zeros(q.shape)
    for i, p in enumerate(positions):
        seen = keys <= p
        if seen.any():
            o[i:i + 1], bound[i:i + 1] = attend(q[i:i + 1], k[seen], v[seen], q.shape[2] ** -0.5)
    return o, bound


@pytest.mark.parametrize("n,d", TILES)
@pytest.mark.parametrize("gone", [(0,), (1,), (4, 5), (6,), (0, 1, 2, 3, 4, 5)])
def test_cache_tiles_blocks_that_are_not_there(stream, n, d, gone):
    """In the first, the second and both places of a tile, the last one, all but the
    last: they count as tokens nobody sees, and block 0, whose scales are NaN, is not
    read for them."""
    queries, lengths = [n, n], [200, 200]
    host, table, q = setup(len(gone), queries, lengths, 4, 2, d)
    table[table == 0] = np.setdiff1d(np.arange(1, len(host.bytes)), table)[0]
    host.scales[0] = np.nan
    asked = table.copy()
    for b in gone:
        asked[0, b], asked[1, b] = -1 - b, len(host.bytes) + b
    got, _ = cache_attention(stream, host, asked, q, queries, lengths)
    keep = np.concatenate([np.arange(b * 32, min(200, b * 32 + 32)) for b in range(7) if b not in gone])
    for s in range(2):
        k, v = (host.values(w, table[s], 200)[keep].astype(np.float64) for w in (0, 1))
        rows = slice(s * n, (s + 1) * n)
        assert_within(got[rows], *attend_at(q[rows], k, v, np.arange(200 - n, 200), keep), f"sequence {s}")


@pytest.mark.parametrize("n,d", TILES)
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("length", [100, 2600])
def test_cache_tiles_scales_that_are_nan(stream, n, d, window, length):
    """They show in the queries that see one of the plane's tokens, and nowhere else."""
    queries, lengths = [n, 1], [length, 33]
    host, table, q = setup(length + window, queries, lengths, 4, 2, d)
    want, in_parts = cache_attention(stream, host, table, q, queries, lengths, window)
    assert in_parts or length < 1000
    for b in set(range(len(host.bytes))) - set(table[0].tolist()) - set(table[1, :2].tolist()):
        host.scales[b] = np.nan  # not in use
    block = (length - n) // BLOCK + 1  # begins behind the first query
    host.scales[table[0, block], 1, 0] = np.nan
    host.scales[table[0, block], 0, 1] = np.nan
    if window:
        host.scales[table[0, 0]] = np.nan
    got, _ = cache_attention(stream, host, table, q, queries, lengths, window)
    nan = np.zeros(got.shape, bool)
    at = np.arange(length - n, length)
    first = np.maximum(at - window + 1, 0) if window else np.zeros(n, int)
    nan[:n][(at >= block * BLOCK) & (first < (block + 1) * BLOCK)] = True
    if window:
        nan[:n][first < BLOCK] = True
    assert np.isnan(got[nan]).all()
    assert (got.view(np.uint16) == want.view(np.uint16))[~nan].all()


@pytest.mark.parametrize("n,d", TILES)
def test_cache_tiles_past_the_stated_context(stream, n, d):
    queries, lengths = [n, 3], [2000, 300]
    host, table, q = setup(9, queries, lengths, 4, 2, d)
    for stated in (1, 64, 1100):
        got, _ = cache_attention(stream, host, table, q, queries, lengths, max_context=stated)
        assert_within(got, *expected(host, table, q, queries, lengths))


@pytest.mark.parametrize("d", [40, 64, 128, 256])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_prompts_in_parts_not_finite_where_not_seen(stream, d, bad):
    """Values and keys that are not finite, in every part, behind the queries' positions
    and before their windows: the queries that do not see them keep every bit."""
    queries, keys, window = [9, 3], [3000, 2500], 700
    rng = np.random.default_rng(d)
    q = rng.standard_normal((12, 4, d)).astype(np.float16)
    k, v = (rng.standard_normal((5500, 2, d)).astype(np.float16) for _ in range(2))
    for w in (0, window):
        want, in_parts = prompt_attention(stream, q, k, v, queries, keys, w)
        assert in_parts
        kb, vb = k.copy(), v.copy()
        seen = np.zeros((12, 5500), bool)
        for row, p in [(i, 2991 + i) for i in range(9)] + [(9 + i, 3000 + 2497 + i) for i in range(3)]:
            start = 0 if row < 9 else 3000
            seen[row, max(start, p - w + 1 if w else start):p + 1] = True
        at = np.array([2993, 2999, 5498, 5499] + ([0, 640, 1500, 2290, 2299, 3000, 4100, 4790] if w else []))
        vb[at, 0, d // 2] = bad
        kb[at, 1] = np.nan
        got, _ = prompt_attention(stream, q, kb, vb, queries, keys, w)
        touched = np.zeros(got.shape, bool)
        touched[:, :2, d // 2] = seen[:, at].any(1)[:, None]
        touched[:, 2:] = seen[:, at].any(1)[:, None, None]
        assert (got.view(np.uint16) == want.view(np.uint16))[~touched].all()
        assert not np.isfinite(got[touched]).any()


# --- each key's weight --------------------------------------------------------------
# Queries of zeros weigh all keys they see alike, 1 / t.  A value that is one in a
# dimension of one key and zero elsewhere then gives 1 / t if the key counts once, 0 if it
# is lost.  Weights are powers of two, their sum over t keys is off by t 2^-23 of it
# at most, its reciprocal and the product by 2^-22, the output by 2^-11.


def single_keys(n, t, window, kv_heads, group, d, keys):
    """Outputs where key keys[h, x] alone is one in dimension x of key head h."""
    at = np.arange(t - n, t)[:, None, None]
    first = np.maximum(at - window + 1, 0) if window else np.zeros_like(at)
    seen = (keys[None] <= at) & (keys[None] >= first)
    return (seen / (at - first + 1)).repeat(group, 1)


def assert_single(got, want, t):
    assert_within(got, want, want * (2.0**-11 + (t + 4) * 2.0**-23) + 2.0**-25)


def key_sets(t, kv_heads, d):
    """Every key once."""
    every = np.arange(-(-t // (kv_heads * d)) * kv_heads * d) % t
    return every.reshape(-1, kv_heads, d)


@pytest.mark.parametrize("n,t,d,heads,kv_heads", [(1, 5000, 128, 4, 2), (70, 3000, 64, 4, 2), (130, 1500, 40, 2, 2),
                                                  (5, 2500, 256, 2, 2), (33, 400, 128, 128, 4)])
@pytest.mark.parametrize("window", [0, 1000])
def test_prompts_each_key_counts_once(stream, n, t, d, heads, kv_heads, window):
    rng = np.random.default_rng(t)
    q = np.zeros((n, heads, d), np.float16)
    k = rng.standard_normal((t, kv_heads, d)).astype(np.float16)
    for keys in key_sets(t, kv_heads, d):
        v = np.zeros((t, kv_heads, d), np.float16)
        v[keys, np.arange(kv_heads)[:, None], np.arange(d)] = 1
        got, _ = prompt_attention(stream, q, k, v, [n], [t], window)
        assert_single(got, single_keys(n, t, window, kv_heads, heads // kv_heads, d, keys), t)


@pytest.mark.parametrize("n,t,d,heads,kv_heads", [(1, 5000, 128, 4, 2), (3, 700, 64, 4, 2), (1, 2500, 256, 2, 2),
                                                  (20, 3000, 64, 4, 2), (60, 3000, 64, 4, 2), (40, 1500, 256, 4, 2),
                                                  (70, 500, 96, 4, 2)])
@pytest.mark.parametrize("window", [0, 1000])
def test_cache_each_key_counts_once(stream, n, t, d, heads, kv_heads, window):
    rng = np.random.default_rng(t)
    blocks = -(-t // BLOCK)
    host = Cache(blocks, kv_heads, d, rng)
    host.scales[..., 1] = 1.0
    table = rng.permutation(blocks).astype(np.int32)[None]
    q = np.zeros((n, heads, d), np.float16)
    for keys in key_sets(t, kv_heads, d):
        host.bytes[:, :, 1] = 128
        for h in range(kv_heads):
            host.bytes[table[0, keys[h] // BLOCK], h, 1, host.index[1][keys[h] % BLOCK, np.arange(d)]] = 129
        got, _ = cache_attention(stream, host, table, q, [n], [t], window)
        assert_single(got, single_keys(n, t, window, kv_heads, heads // kv_heads, d, keys), t)
