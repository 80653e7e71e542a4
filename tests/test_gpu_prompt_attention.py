"""Attention of packed prompts against the 64-bit oracle: lengths around the
tiles' edges, empty sequences, queries that see nothing, grouped heads, head
sizes that are no tile's, windows, keys divided into parts, strides and odd
addresses, values that are not finite in keys a query does not see, other
streams, graphs.  The bound is the oracle's, derived from the number formats."""

from __future__ import annotations

import numpy as np
import pytest

from attention_oracle import assert_within, attend
from mote_amd import ops
from mote_amd.device import DeviceBuffer, Stream
from mote_amd.hip_runtime import HipRuntime

pytestmark = pytest.mark.gpu

SENTINEL = 0x7A


def offsets(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def tensors(seed, queries, keys, heads, kv_heads, d, spread=1.5):
    rng = np.random.default_rng(seed)
    q = (rng.standard_normal((sum(queries), heads, d)) * spread).astype(np.float16)
    k = rng.standard_normal((sum(keys), kv_heads, d)).astype(np.float16)
    v = rng.standard_normal((sum(keys), kv_heads, d)).astype(np.float16)
    return q, k, v


def spaced(x, stride, skip=0):
    """Rows of x `stride` elements apart, from element `skip` on."""
    flat = np.full(skip + max(len(x), 1) * stride, 0x7E00, np.uint16)  # NaN between
    rows = flat[skip:].reshape(-1, stride)
    rows[: len(x), : x[0].size if len(x) else 0] = x.reshape(len(x), -1).view(np.uint16)
    return flat


class Call:
    """One call's device buffers."""

    def __init__(self, q, k, v, queries, keys, causal=True, window=0, strides=None, skip=0, own_keys=False):
        self.heads, self.kv_heads, self.d = q.shape[1], k.shape[1], q.shape[2]
        wide = (self.heads * self.d, self.kv_heads * self.d, self.kv_heads * self.d, self.heads * self.d)
        self.strides, self.skip = strides or wide, skip
        self.q, self.k, self.v = (DeviceBuffer.from_array(spaced(x, s, skip))
                                  for x, s in zip((q, k, v), self.strides))
        self.rows = len(q)
        self.out_size = (skip + max(self.rows, 1) * self.strides[3]) * 2
        self.out = DeviceBuffer.from_array(np.full(self.out_size, SENTINEL, np.uint8))
        self.at = DeviceBuffer.from_array(offsets(queries))
        self.key_at = None if own_keys else DeviceBuffer.from_array(offsets(keys))
        self.sizes = (len(queries), sum(queries), sum(keys), max(keys, default=0), self.heads, self.kv_heads, self.d)
        self.need = ops.prompt_attention_workspace(*self.sizes)
        self.work = DeviceBuffer(self.need)
        self.mask = dict(causal=causal, window=window)
        self.scale = self.d ** -0.5

    def run(self, stream, out=None):
        e = 2 * self.skip
        ops.prompt_attention_f16(
            self.q.ptr + e, self.k.ptr + e, self.v.ptr + e, out or self.out.ptr + e, self.at.ptr,
            self.key_at.ptr if self.key_at else None, *self.sizes, self.scale, self.work.ptr, self.need, stream,
            strides=self.strides, **self.mask)

    def result(self, stream):
        stream.synchronize()
        rows = self.out.download(np.uint16)[self.skip:].reshape(-1, self.strides[3])[: self.rows]
        gap = rows[:, self.heads * self.d:]
        assert (gap == SENTINEL * 0x0101).all(), "written between the rows"
        return rows[:, : self.heads * self.d].copy().view(np.float16).reshape(self.rows, self.heads, self.d)


def expected(q, k, v, queries, keys, scale, causal=True, window=0):
    o, b = np.zeros(q.shape), np.zeros(q.shape)
    i = j = 0
    for n, t in zip(queries, keys):
        o[i:i + n], b[i:i + n] = attend(q[i:i + n], k[j:j + t], v[j:j + t], scale, causal, window)
        i, j = i + n, j + t
    return o, b


def check(stream, seed, queries, keys, heads, kv_heads, d, spread=1.5, **how):
    q, k, v = tensors(seed, queries, keys, heads, kv_heads, d, spread)
    call = Call(q, k, v, queries, keys, **how)
    call.run(stream)
    mask = {x: how[x] for x in ("causal", "window") if x in how}
    o, bound = expected(q, k, v, queries, keys, call.scale, **mask)
    assert_within(call.result(stream), o, bound)
    return call


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 300])
def test_one_sequence(stream, n):
    check(stream, n, [n], [n], 4, 2, 64, own_keys=True)


@pytest.mark.parametrize("d", [8, 16, 40, 64, 72, 80, 96, 104, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_head_sizes(stream, d, causal):
    check(stream, d, [70, 5], [90, 140], 2, 1, d, causal=causal)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (7, 1), (10, 2), (16, 16)])
def test_head_groups(stream, heads, kv_heads):
    check(stream, heads, [40, 100], [40, 130], heads, kv_heads, 64)


@pytest.mark.parametrize("queries,keys", [
    ([0, 5, 0, 1, 130, 0], [3, 5, 0, 40, 130, 9]),        # sequences without queries, or nothing at all
    ([1] * 70 + [50], [1] * 70 + [50]),                   # more sequences than a wave looks up at once
    ([0, 3, 0, 200] * 40, [2, 3, 0, 200] * 40),
    ([5, 90, 3], [2, 40, 0]),                             # fewer keys than queries: the first see nothing
    ([128, 256, 64], [128, 256, 64]),                     # whole tiles
])
def test_packed(stream, queries, keys):
    check(stream, len(queries), queries, keys, 2, 1, 64)


@pytest.mark.parametrize("how", [dict(), dict(causal=False), dict(window=1), dict(window=33), dict(window=64)])
def test_many_workgroups(stream, how):
    """More than a thousand, which take shorter tiles of keys."""
    queries = [1, 31, 32, 33, 0, 64, 65, 130]
    check(stream, 12, queries, [1, 40, 32, 95, 5, 64, 65, 200], 128, 4, 128, **how)


def test_many_workgroups_not_finite_where_not_seen(stream):
    queries = [130, 60, 60, 60, 60, 60, 60]
    q, k, v = tensors(13, queries, queries, 128, 2, 128)
    clean = Call(q, k, v, queries, queries)
    clean.run(stream)
    want = clean.result(stream)
    k[100, 0], v[101, 0, 3], v[180, 1, 5] = np.nan, np.inf, np.nan
    call = Call(q, k, v, queries, queries)
    call.run(stream)
    got = call.result(stream)
    touched = np.zeros(got.shape, bool)
    touched[100:130, :64] = True
    touched[101:130, :64, 3] = True
    touched[180:190, 64:, 5] = True
    assert (got.view(np.uint16) == want.view(np.uint16))[~touched].all()
    assert np.isnan(got[touched]).all()


@pytest.mark.parametrize("count", [4097, 70000])
def test_very_many_sequences(stream, count):
    """Of one token each (whose attention is its value) and now and then five: three
    steps of the look-up, and more tiles than one launch has room for."""
    rng = np.random.default_rng(count)
    lengths = np.ones(count, np.int64)
    lengths[rng.integers(0, count, 50)] = 5
    q, k, v = tensors(count, lengths.tolist(), lengths.tolist(), 1, 1, 8)
    call = Call(q, k, v, lengths.tolist(), lengths.tolist(), own_keys=True)
    call.run(stream)
    got = call.result(stream)
    at = np.concatenate([[0], np.cumsum(lengths)])[:-1]
    single = at[lengths == 1]
    assert (got[single].view(np.uint16) == v[single].view(np.uint16)).all()
    for a in at[lengths == 5]:
        o, bound = attend(q[a:a + 5], k[a:a + 5], v[a:a + 5], call.scale)
        assert_within(got[a:a + 5], o, bound)


@pytest.mark.parametrize("window", [1, 2, 17, 63, 64, 65, 100, 129, 299, 300, 301, 1 << 40])
def test_windows(stream, window):
    check(stream, 5, [300, 40], [300, 333], 2, 2, 64, window=window)


@pytest.mark.parametrize("queries,keys,d", [([1], [3000], 128), ([9, 2], [1500, 2600], 64), ([130], [2500], 96),
                                            ([3, 1], [2, 4000], 256)])
@pytest.mark.parametrize("window", [0, 700])
def test_keys_in_parts(stream, queries, keys, d, window):
    call = check(stream, d, queries, keys, 4, 2, d, window=window)
    assert call.need > 0


def test_scores_that_grow_along_the_keys(stream):
    """The running maximum grows in every tile, by more and by less than what
    rescales the sums, and falls again."""
    rng = np.random.default_rng(3)
    n, d = 400, 64
    q = np.abs(rng.standard_normal((n, 1, d))).astype(np.float16)
    k = np.abs(rng.standard_normal((n, 1, d)))
    k *= np.concatenate([np.linspace(0.01, 6, 250), np.linspace(6, 0.01, 150)])[:, None, None]
    v = rng.standard_normal((n, 1, d)).astype(np.float16)
    k = k.astype(np.float16)
    call = Call(q, k, v, [n], [n])
    call.run(stream)
    o, bound = expected(q, k, v, [n], [n], call.scale)
    assert_within(call.result(stream), o, bound)


def test_strides_and_odd_addresses(stream):
    """Rows apart, from an address on no grid but the element's."""
    for skip, gaps in ((0, (8, 16, 24, 8)), (1, (3, 5, 7, 9)), (3, (1, 0, 2, 1))):
        d, heads, kv_heads = 72, 4, 2
        strides = tuple(w * d + g for w, g in zip((heads, kv_heads, kv_heads, heads), gaps))
        check(stream, skip, [130, 7], [130, 150], heads, kv_heads, d, strides=strides, skip=skip)


def test_rows_shared_by_all_keys(stream):
    """A stride of 0: the same key and value everywhere."""
    rng = np.random.default_rng(1)
    q = rng.standard_normal((50, 2, 64)).astype(np.float16)
    k, v = (rng.standard_normal((1, 1, 64)).astype(np.float16) for _ in range(2))
    call = Call(q, np.repeat(k, 50, 0), np.repeat(v, 50, 0), [50], [50])
    call.strides = (128, 0, 0, 128)
    call.run(stream)
    assert_within(call.result(stream), np.broadcast_to(v.astype(np.float64), q.shape),
                  np.full(q.shape, 2.0**-10 * np.abs(v).max() * 2))


def test_output_over_the_queries(stream):
    q, k, v = tensors(4, [200], [200], 2, 1, 64)
    call = Call(q, k, v, [200], [200])
    call.run(stream)
    want = call.result(stream)
    call.run(stream, out=call.q.ptr)
    stream.synchronize()
    assert (call.q.download(np.uint16).reshape(want.shape) == want.view(np.uint16)).all()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("d", [40, 128])
@pytest.mark.parametrize("what", ["k", "v", "both"])
def test_not_finite_where_not_seen(stream, bad, d, what):
    """A key or value that is not finite changes the queries that see it and no
    other: those before it, those past its window, other sequences, and other
    heads keep every bit."""
    queries, window = [150, 60], 50
    q, k, v = tensors(6, queries, queries, 4, 2, d)
    clean = Call(q, k, v, queries, queries, window=window)
    clean.run(stream)
    want = clean.result(stream)
    at = [70, 149, 150 + 59]
    for j in at:
        if what != "v":
            k[j, 0] = bad
        if what != "k":
            v[j, 0, d // 2] = bad
    call = Call(q, k, v, queries, queries, window=window)
    call.run(stream)
    got = call.result(stream)
    touched = np.zeros(got.shape, bool)
    for j in at:
        last = 150 if j < 150 else 210
        touched[j:min(j + window, last), :2] = True
    if what == "v":
        only = np.zeros_like(touched)
        only[..., d // 2] = True
        touched &= only
    assert (got.view(np.uint16) == want.view(np.uint16))[~touched].all()
    if what != "k" and not np.isnan(bad):
        assert not np.isfinite(got[70:120, :2, d // 2]).any()
    if np.isnan(bad):
        assert np.isnan(got[touched]).all()


def test_not_finite_between_the_sequences_and_past_the_end(stream):
    """Rows of other sequences lie in the same tiles."""
    queries, keys = [20, 30], [20, 30]
    q, k, v = tensors(8, queries, keys, 2, 1, 64)
    clean = Call(q, k, v, queries, keys)
    clean.run(stream)
    want = clean.result(stream)
    k[20:], v[20:] = np.nan, np.inf
    call = Call(q, k, v, queries, keys)
    call.run(stream)
    assert (call.result(stream)[:20].view(np.uint16) == want[:20].view(np.uint16)).all()


def test_large_and_small_scores(stream):
    check(stream, 9, [100], [150], 2, 1, 64, spread=300.0)
    check(stream, 9, [100], [150], 2, 1, 64, spread=1e-4)


def test_repeats_and_streams_agree(stream):
    q, k, v = tensors(10, [9, 200], [2000, 200], 4, 2, 64)
    call = Call(q, k, v, [9, 200], [2000, 200])
    call.run(stream)
    want = call.result(stream).copy()
    other = Stream()
    for s in (stream, other, stream):
        call.out.upload(np.full(call.out_size, SENTINEL, np.uint8))
        call.run(s)
        assert (call.result(s).view(np.uint16) == want.view(np.uint16)).all()
    other.close()


def test_graph(stream):
    hip = HipRuntime()
    q, k, v = tensors(11, [9, 20], [1500, 70], 4, 2, 64)
    call = Call(q, k, v, [9, 20], [1500, 70])
    call.run(stream)
    want = call.result(stream).copy()
    graph = hip.capture(stream, lambda: call.run(stream))
    for i in range(3):
        call.out.upload(np.full(call.out_size, SENTINEL, np.uint8))
        hip.launch_graph(graph, stream)
        assert (call.result(stream).view(np.uint16) == want.view(np.uint16)).all()
        call.run(stream)
        stream.synchronize()
    hip.destroy_graph(graph)
