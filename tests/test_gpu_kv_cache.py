"""The 8-bit cache: what append writes and read gives back, byte for byte
against the f32 steps that define them, and attention over it against the 64-bit
oracle on what the bytes stand for."""

from __future__ import annotations

import numpy as np
import pytest

from attention_oracle import BLOCK, Cache, assert_within, attend, padded
from mote_amd import ops
from mote_amd.device import DeviceBuffer, Stream
from mote_amd.hip_runtime import HipRuntime

pytestmark = pytest.mark.gpu


def offsets(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def ints(x):
    return np.asarray(x, np.int32)


def tables(rng, sequences, blocks, pool):
    return rng.permutation(pool)[: sequences * blocks].reshape(sequences, blocks).astype(np.int32)


class Held:
    """A cache on the device beside the host's."""

    def __init__(self, host: Cache, table):
        self.host, self.table = host, ints(table)
        self.cache = DeviceBuffer.from_array(host.bytes)
        self.scales = DeviceBuffer.from_array(host.scales)
        self.tab = DeviceBuffer.from_array(self.table)

    def append(self, stream, k, v, lengths, positions, strides=None, skip=0):
        heads, d = self.host.heads, self.host.d
        sk, sv = strides or (heads * d, heads * d)
        bufs = []
        for x, s in ((k, sk), (v, sv)):
            flat = np.full(skip + max(len(x), 1) * s, 0x7E00, np.uint16)
            flat[skip:].reshape(-1, s)[: len(x), : heads * d] = x.reshape(len(x), -1).view(np.uint16)
            bufs.append(DeviceBuffer.from_array(flat))
        at, pos = DeviceBuffer.from_array(offsets(lengths)), DeviceBuffer.from_array(ints(positions))
        ops.kv_cache_append_q8(bufs[0].ptr + 2 * skip, bufs[1].ptr + 2 * skip, at.ptr, pos.ptr, self.tab.ptr,
                               self.cache.ptr, self.scales.ptr, len(lengths), sum(lengths), heads, d,
                               self.table.shape[1], len(self.host.bytes), stream, strides=(sk, sv))
        stream.synchronize()
        row = 0
        for s, n in enumerate(lengths):
            for which, x in ((0, k), (1, v)):
                self.host.append(x[row:row + n], which, self.table[s], positions[s])
            row += n

    def read(self, stream, lengths, positions):
        heads, d = self.host.heads, self.host.d
        total = max(sum(lengths), 1)
        out = [DeviceBuffer.from_array(np.full(total * heads * d, 0x7A7A, np.uint16)) for _ in range(2)]
        at, pos = DeviceBuffer.from_array(offsets(lengths)), DeviceBuffer.from_array(ints(positions))
        ops.kv_cache_read_q8_f16(self.cache.ptr, self.scales.ptr, at.ptr, pos.ptr, self.tab.ptr, out[0].ptr,
                                 out[1].ptr, len(lengths), sum(lengths), heads, d, self.table.shape[1],
                                 len(self.host.bytes), stream)
        stream.synchronize()
        return [x.download(np.float16).reshape(total, heads, d) for x in out]

    def check(self):
        """Every byte and every scale equals the host's."""
        got = self.cache.download(np.uint8).reshape(self.host.bytes.shape)
        scales = self.scales.download(np.float32).reshape(self.host.scales.shape)
        assert np.array_equal(scales, self.host.scales, equal_nan=True)
        assert (got == self.host.bytes).all(), np.argwhere(got != self.host.bytes)[0]


def rows(rng, n, heads, d, size=1.0):
    return (rng.standard_normal((n, heads, d)) * size).astype(np.float16)


@pytest.mark.parametrize("d", [8, 32, 40, 64, 96, 128, 200, 256])
def test_append_whole_prompts(stream, d):
    rng = np.random.default_rng(d)
    lengths = [0, 1, 31, 32, 33, 70, 0, 64]
    held = Held(Cache(30, 2, d, rng), tables(rng, 8, 3, 30))
    k, v = rows(rng, sum(lengths), 2, d), rows(rng, sum(lengths), 2, d, 0.1)
    held.append(stream, k, v, lengths, [0] * 8)
    held.check()
    got = held.read(stream, lengths, [0] * 8)
    row = 0
    for s, n in enumerate(lengths):
        for which in (0, 1):
            want = held.host.values(which, held.table[s], n).astype(np.float16)
            assert (got[which][row:row + n].view(np.uint16) == want.view(np.uint16)).all()
        row += n


def test_append_token_by_token(stream):
    """Scales that grow as tokens come, blocks that begin, a sequence that
    pauses: the same bytes as the host's after every step."""
    rng = np.random.default_rng(1)
    held = Held(Cache(9, 3, 72, rng), tables(rng, 3, 3, 9))
    at = [0, 17, 31]
    first = [0, 17, 31]
    k, v = rows(rng, 48, 3, 72), rows(rng, 48, 3, 72)
    held.append(stream, k, v, first, [0, 0, 0])
    for step in range(40):
        now = [1, 1, 0 if step % 5 == 3 else 1]
        size = 1.0 + 0.2 * (step % 7)
        held.append(stream, rows(rng, sum(now), 3, 72, size), rows(rng, sum(now), 3, 72, size), now, at)
        at = [a + n for a, n in zip(at, now)]
        held.check()


def test_append_pieces_join(stream):
    """Prompts in chunks that end inside blocks."""
    rng = np.random.default_rng(2)
    held = Held(Cache(40, 2, 64, rng), tables(rng, 2, 8, 40))
    at = [0, 0]
    for now in ([5, 100], [27, 3], [1, 40], [90, 0], [33, 66]):
        held.append(stream, rows(rng, sum(now), 2, 64), rows(rng, sum(now), 2, 64), now, at)
        at = [a + n for a, n in zip(at, now)]
        held.check()
    # back to an earlier token: the block keeps its scale, later blocks start anew
    at = [40, 65]
    held.append(stream, rows(rng, 60, 2, 64, 0.1), rows(rng, 60, 2, 64, 0.1), [30, 30], at)
    held.check()


def test_append_to_many_sequences(stream):
    """More than a wave looks up at once, most of them with nothing new."""
    rng = np.random.default_rng(17)
    held = Held(Cache(300, 1, 32, rng), tables(rng, 150, 2, 300))
    lengths = [int(n) for n in rng.choice([0, 0, 1, 5, 33], 150)]
    positions = [int(p) for p in rng.integers(0, 31, 150)]
    held.append(stream, rows(rng, sum(lengths), 1, 32), rows(rng, sum(lengths), 1, 32), lengths, positions)
    held.check()


def test_append_zeros_and_extremes(stream):
    rng = np.random.default_rng(3)
    held = Held(Cache(6, 1, 64, rng), tables(rng, 1, 6, 6))
    x = rows(rng, 192, 1, 64)
    x[:32] = 0                                   # an all-zero block, then tokens that join none
    x[32:64] = np.float16(6e-8)                  # the smallest subnormal
    x[64:96] *= np.float16(65504 / 8)            # the largest
    x[64, 0, 0] = np.float16(-65504)
    x[96:128] = np.float16(-0.0)
    held.append(stream, x, x, [192], [0])
    held.check()
    held.append(stream, x[130:140], x[:10], [10], [5])  # joins the all-zero block
    held.check()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_append_not_finite(stream, bad):
    """The plane that takes one reads as NaN until its block begins anew; the
    other planes are as ever."""
    rng = np.random.default_rng(4)
    held = Held(Cache(4, 2, 64, rng), tables(rng, 1, 4, 4))
    k, v = rows(rng, 70, 2, 64), rows(rng, 70, 2, 64)
    k[40, 1, 3] = bad
    held.append(stream, k, v, [70], [0])
    held.check()
    held.append(stream, v[:1], k[:1], [1], [45])
    held.check()
    got = held.read(stream, [70], [0])
    assert np.isnan(got[0][32:64, 1]).all() and np.isfinite(got[0][:32]).all() and np.isfinite(got[0][32:64, 0]).all()
    assert np.isfinite(got[1]).all()
    held.append(stream, v[:20], k[:20], [20], [32])
    held.check()
    assert np.isfinite(held.read(stream, [52], [0])[0]).all()


def test_append_strides_and_odd_addresses(stream):
    rng = np.random.default_rng(5)
    for skip, gap in ((0, 8), (1, 3), (5, 0)):
        held = Held(Cache(8, 2, 40, rng), tables(rng, 2, 4, 8))
        k, v = rows(rng, 90, 2, 40), rows(rng, 90, 2, 40)
        held.append(stream, k, v, [50, 40], [0, 13], strides=(80 + gap, 80 + 2 * gap), skip=skip)
        held.check()


def test_tokens_past_the_table_and_blocks_that_are_not_there(stream):
    rng = np.random.default_rng(6)
    table = tables(rng, 2, 3, 8)
    table[0, 1] = -1
    table[1, 0] = 8
    held = Held(Cache(8, 1, 32, rng), table)
    before = held.host.bytes.copy(), held.host.scales.copy()
    held.append(stream, rows(rng, 300, 1, 32), rows(rng, 300, 1, 32), [130, 170], [0, 0])
    got = held.cache.download(np.uint8).reshape(before[0].shape)
    scales = held.scales.download(np.float32).reshape(before[1].shape)
    assert (got == held.host.bytes).all() and (scales == held.host.scales).all()
    valid = {int(b) for b in table.ravel() if 0 <= b < 8}
    for b in set(range(8)) - valid:
        assert (got[b] == before[0][b]).all()
    out = held.read(stream, [130, 170], [0, 0])
    missing = np.concatenate([np.arange(32, 64), np.arange(96, 130), 130 + np.arange(32), 130 + np.arange(96, 170)])
    assert (out[0].view(np.uint16)[missing] == 0x7A7A).all()  # left as they were


def test_read_from_inside_a_block(stream):
    rng = np.random.default_rng(7)
    held = Held(Cache(10, 2, 72, rng), tables(rng, 2, 5, 10))
    got = held.read(stream, [70, 3], [45, 30])
    for which in (0, 1):
        a = held.host.values(which, held.table[0], 115)[45:]
        b = held.host.values(which, held.table[1], 33)[30:]
        want = np.concatenate([a, b]).astype(np.float16)
        assert (got[which].view(np.uint16) == want.view(np.uint16)).all()


# --- attention over the cache -----------------------------------------------------


class Attend:
    def __init__(self, held, q, queries, lengths, window=0, spread=0, skip=0, max_context=None, single=False):
        self.heads, self.d, self.rows = q.shape[1], q.shape[2], len(q)
        self.held, self.window, self.skip = held, window, skip
        self.stride = self.heads * self.d + spread
        flat = np.full(skip + max(self.rows, 1) * self.stride, 0x7E00, np.uint16)
        flat[skip:].reshape(-1, self.stride)[: self.rows, : self.heads * self.d] = q.reshape(self.rows, -1).view(np.uint16)
        self.q = DeviceBuffer.from_array(flat)
        self.out = DeviceBuffer.from_array(np.full(flat.size, 0x7A7A, np.uint16))
        self.at = None if single else DeviceBuffer.from_array(offsets(queries))
        self.lengths = DeviceBuffer.from_array(ints(lengths))
        self.sizes = (len(queries), self.rows, max(queries, default=0), max_context or max(lengths), self.heads,
                      held.host.heads, self.d)
        self.need = ops.cache_attention_workspace(*self.sizes)
        self.work = DeviceBuffer(self.need)
        self.scale = self.d ** -0.5

    def run(self, stream):
        e = 2 * self.skip
        ops.cache_attention_q8_f16(
            self.q.ptr + e, self.held.cache.ptr, self.held.scales.ptr, self.at.ptr if self.at else None,
            self.lengths.ptr, self.held.tab.ptr, self.out.ptr + e, *self.sizes, self.held.table.shape[1],
            len(self.held.host.bytes), self.scale, self.work.ptr, self.need, stream, window=self.window,
            strides=(self.stride, self.stride))

    def result(self, stream):
        stream.synchronize()
        rows = self.out.download(np.uint16)[self.skip:].reshape(-1, self.stride)[: self.rows]
        assert (rows[:, self.heads * self.d:] == 0x7A7A).all(), "written between the rows"
        return rows[:, : self.heads * self.d].copy().view(np.float16).reshape(self.rows, self.heads, self.d)


def setup(seed, queries, lengths, heads, kv_heads, d, spread=1.5):
    rng = np.random.default_rng(seed)
    blocks = max(-(-max(lengths) // BLOCK), 1)
    pool = len(lengths) * blocks + 2
    held = Held(Cache(pool, kv_heads, d, rng), tables(rng, len(lengths), blocks, pool))
    q = (rng.standard_normal((sum(queries), heads, d)) * spread).astype(np.float16)
    return held, q


def expected(held, q, queries, lengths, window=0):
    o, b = np.zeros(q.shape), np.zeros(q.shape)
    row = 0
    for s, (n, t) in enumerate(zip(queries, lengths)):
        k, v = (held.host.values(w, held.table[s], t).astype(np.float64) for w in (0, 1))
        o[row:row + n], b[row:row + n] = attend(q[row:row + n], k, v, q.shape[2] ** -0.5, True, window)
        row += n
    return o, b


def check(stream, seed, queries, lengths, heads, kv_heads, d, window=0, spread=1.5, **how):
    held, q = setup(seed, queries, lengths, heads, kv_heads, d, spread)
    call = Attend(held, q, queries, lengths, window, **how)
    call.run(stream)
    o, bound = expected(held, q, queries, lengths, window)
    assert_within(call.result(stream), o, bound)
    return call


@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 64, 127, 128, 129, 255, 256, 257, 700])
def test_one_token(stream, length):
    check(stream, length, [1], [length], 8, 2, 128, single=length % 2 == 0)


@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 96, 104, 128, 136, 160, 192, 200, 224, 256])
@pytest.mark.parametrize("n", [1, 5, 13, 40])
def test_head_sizes(stream, d, n):
    check(stream, d, [n, n], [70, 300], 8, 2, d)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 1), (16, 1), (17, 1), (40, 1), (6, 3), (8, 8)])
def test_head_groups(stream, heads, kv_heads):
    check(stream, heads, [1, 1], [200, 31], heads, kv_heads, 64)
    check(stream, heads, [3, 2], [200, 31], heads, kv_heads, 64)


@pytest.mark.parametrize("queries,lengths", [
    ([1, 1, 1, 1], [0, 1, 500, 32]),                # a sequence that holds nothing: zeros
    ([0, 4, 0, 1, 70], [9, 4, 0, 300, 70]),         # ragged queries, some sequences without
    ([5, 90], [2, 40]),                             # more queries than tokens: the first see nothing
    ([1] * 100, list(range(1, 101))),
    ([130, 7], [400, 1000]),                        # a chunk of a prompt
])
def test_ragged(stream, queries, lengths):
    check(stream, len(queries), queries, lengths, 4, 2, 64)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 299, 300, 1 << 50])
@pytest.mark.parametrize("n", [1, 6, 40])
def test_windows(stream, window, n):
    check(stream, window % 1000, [n, n], [300, 77], 4, 2, 64, window=window)


@pytest.mark.parametrize("n,d", [(1, 128), (1, 256), (4, 64), (30, 96)])
@pytest.mark.parametrize("window", [0, 1500])
def test_long_contexts_in_parts(stream, n, d, window):
    call = check(stream, d, [n, n], [5000, 2500], 4, 2, d, window=window)
    assert call.need > 0


def test_context_past_the_stated_most(stream):
    """max_context only divides the work: a longer context is still read whole."""
    check(stream, 3, [1, 2], [2000, 300], 4, 2, 64, max_context=64)


def test_strides_and_odd_addresses(stream):
    for skip, spread in ((0, 8), (1, 3), (7, 0)):
        check(stream, skip, [3, 1], [100, 50], 4, 2, 72, spread=spread, skip=skip)


def test_blocks_that_are_not_there(stream):
    """They count as tokens nobody sees."""
    held, q = setup(12, [1, 2], [200, 200], 4, 2, 64)
    held.table[0, 2], held.table[1, 0] = -1, len(held.host.bytes)
    held.tab.upload(held.table)
    call = Attend(held, q, [1, 2], [200, 200])
    call.run(stream)
    got = call.result(stream)
    for s, (row, n, gone) in enumerate(((0, 1, 2), (1, 2, 0))):
        keep = np.concatenate([np.arange(b * 32, min(200, b * 32 + 32)) for b in range(7) if b != gone])
        table = np.where(np.arange(7) == gone, 0, held.table[s])
        k, v = (held.host.values(w, table, 200)[keep].astype(np.float64) for w in (0, 1))
        o, bound = attend(q[row:row + n], k, v, call.scale)
        assert_within(got[row:row + n], o, bound)


def test_scales_that_are_nan(stream):
    """A NaN plane shows in the queries that see one of its tokens, in no other
    query, head or sequence; what follows a sequence's last token in its block, and
    blocks past it, are not seen."""
    queries, lengths = [40, 1], [100, 33]
    held, q = setup(13, queries, lengths, 4, 2, 64)
    call = Attend(held, q, queries, lengths)
    call.run(stream)
    want = call.result(stream)
    used = {int(b) for s, t in enumerate(lengths) for b in held.table[s, : -(-t // 32)]}
    for b in set(range(len(held.host.bytes))) - used:
        held.host.scales[b] = np.nan
    held.host.scales[held.table[0, 2], 1, 0] = np.nan  # keys of tokens 64 .. 95, head 1
    held.host.scales[held.table[0, 3], 0, 1] = np.nan  # values of tokens 96 .., head 0
    held.scales.upload(held.host.scales)
    call = Attend(held, q, queries, lengths)
    call.run(stream)
    got = call.result(stream)
    nan = np.zeros(got.shape, bool)
    nan[4:40, 2:] = True  # positions 64 ..
    nan[36:40, :2] = True  # positions 96 ..
    assert np.isnan(got[nan]).all()
    assert (got.view(np.uint16) == want.view(np.uint16))[~nan].all()


def test_scores_that_grow_along_the_context(stream):
    rng = np.random.default_rng(14)
    held, q = setup(14, [1, 3], [900, 600], 4, 1, 64)
    q[:] = np.abs(q)
    order = np.argsort([list(held.table.ravel()).index(b) if b in held.table else 0 for b in range(len(held.host.bytes))])
    held.host.bytes[:, :, 0] = rng.integers(128, 256, held.host.bytes[:, :, 0].shape)
    held.host.scales[order, :, 0] = np.linspace(1e-4, 0.1, len(order), dtype=np.float32)[:, None]
    held.cache.upload(held.host.bytes)
    held.scales.upload(held.host.scales)
    call = Attend(held, q, [1, 3], [900, 600])
    call.run(stream)
    o, bound = expected(held, q, [1, 3], [900, 600])
    assert_within(call.result(stream), o, bound)


def test_offsets_past_32_bits(stream):
    """Blocks beyond 4 GiB: append, read and attend there."""
    rng = np.random.default_rng(15)
    kv_heads, d = 8, 256
    plane = 2 * kv_heads * BLOCK * padded(d)
    blocks = (5 << 30) // plane
    table = ints([[blocks - 1, blocks - 3, 2, blocks - 2]])
    small = Cache(4, kv_heads, d)
    cache, scales = DeviceBuffer(blocks * plane), DeviceBuffer(blocks * kv_heads * 2 * 4)
    k, v = rows(rng, 110, kv_heads, d), rows(rng, 110, kv_heads, d)
    for which, x in ((0, k), (1, v)):
        small.append(x, which, [0, 1, 2, 3], 0)
    kb, vb, tab = (DeviceBuffer.from_array(x) for x in (k, v, table))
    at, pos, n = (DeviceBuffer.from_array(ints(x)) for x in ([0, 110], [0], [110]))
    ops.kv_cache_append_q8(kb.ptr, vb.ptr, at.ptr, pos.ptr, tab.ptr, cache.ptr, scales.ptr, 1, 110, kv_heads, d, 4,
                           blocks, stream)
    back = [DeviceBuffer(k.nbytes) for _ in range(2)]
    ops.kv_cache_read_q8_f16(cache.ptr, scales.ptr, at.ptr, pos.ptr, tab.ptr, back[0].ptr, back[1].ptr, 1, 110,
                             kv_heads, d, 4, blocks, stream)
    q = rows(rng, 1, 16, d)
    qb, out = DeviceBuffer.from_array(q), DeviceBuffer(q.nbytes)
    need = ops.cache_attention_workspace(1, 1, 1, 110, 16, kv_heads, d)
    work = DeviceBuffer(need)
    ops.cache_attention_q8_f16(qb.ptr, cache.ptr, scales.ptr, None, n.ptr, tab.ptr, out.ptr, 1, 1, 1, 110, 16, kv_heads,
                               d, 4, blocks, d ** -0.5, work.ptr, need, stream)
    stream.synchronize()
    held = [small.values(w, [0, 1, 2, 3], 110) for w in (0, 1)]
    for w in (0, 1):
        got = back[w].download(np.uint16).reshape(k.shape)
        assert (got == held[w].astype(np.float16).view(np.uint16)).all()
    o, bound = attend(q, held[0].astype(np.float64), held[1].astype(np.float64), d ** -0.5)
    assert_within(out.download(np.float16).reshape(q.shape), o, bound)


def test_repeats_streams_and_graphs_agree(stream):
    hip = HipRuntime()
    held, q = setup(16, [1, 3], [3000, 600], 8, 2, 128)
    call = Attend(held, q, [1, 3], [3000, 600])
    call.run(stream)
    want = call.result(stream).copy()
    other = Stream()
    for s in (other, stream):
        call.out.upload(np.full(call.out.nbytes // 2, 0x7A7A, np.uint16))
        call.run(s)
        assert (call.result(s).view(np.uint16) == want.view(np.uint16)).all()
    other.close()
    graph = hip.capture(stream, lambda: call.run(stream))
    for _ in range(3):
        call.out.upload(np.full(call.out.nbytes // 2, 0x7A7A, np.uint16))
        hip.launch_graph(graph, stream)
        assert (call.result(stream).view(np.uint16) == want.view(np.uint16)).all()
        call.run(stream)
        stream.synchronize()
    hip.destroy_graph(graph)


def test_graph_replayed_with_other_lengths(stream):
    """Only the sizes given by the host divide the work: what a graph holds stays
    right as the lengths on the device change."""
    hip = HipRuntime()
    held, q = setup(18, [1, 1, 1], [2000, 1500, 700], 8, 2, 64)
    call = Attend(held, q, [1, 1, 1], [2000, 1500, 700], single=True)
    call.run(stream)
    call.result(stream)
    graph = hip.capture(stream, lambda: call.run(stream))
    for lengths in ([2000, 1500, 700], [1, 33, 0], [64, 1999, 1000]):
        call.lengths.upload(ints(lengths))
        call.run(stream)
        eager = call.result(stream).copy()
        call.out.upload(np.full(call.out.nbytes // 2, 0x7A7A, np.uint16))
        hip.launch_graph(graph, stream)
        assert (call.result(stream).view(np.uint16) == eager.view(np.uint16)).all()
        o, bound = expected(held, q, [1, 1, 1], lengths)
        assert_within(eager, o, bound)
    hip.destroy_graph(graph)
