"""Routing, its plan and the experts' products against 64 bits.

Products are exact in 32 bits (tests/test_gpu_mx_linear.py says why), so what is left is
* gate/up: silu by the device's exponential and one rounding.  e^-g of |g| up to 88 is
  good to 2^-21 + |g| 2^-23 (its argument times log2 e is rounded once), the quotient and two
  products to 2^-23 each: 2^-15 covers them up to |g| = 600, where silu is g or nothing;
  and half a step of binary16, 2^-11, or 2^-25 under its normal numbers.
* down: terms weight x product added in 32 bits, each addition and product good to
  2^-24 of the sum of the sizes: (top + 1) 2^-23, then half a step of binary16."""

from __future__ import annotations

import numpy as np
import pytest

import mx_oracle as mx
from mote_amd import ops
from mote_amd.device import DeviceBuffer
from mote_amd.hip_runtime import HipRuntime

pytestmark = pytest.mark.gpu

ROUTE = {np.float16: ops.route_experts_f16, np.float32: ops.route_experts_f32}


def route(stream, logits, bias, top, score, **more):
    tokens, experts = logits.shape
    x = DeviceBuffer.from_array(logits)
    b = DeviceBuffer.from_array(np.asarray(bias, np.float32)) if bias is not None else None
    ids = DeviceBuffer.from_array(np.full(tokens * top + 16, 77, np.int32))
    weights = DeviceBuffer.from_array(np.full(tokens * top + 16, 77, np.float32))
    ROUTE[logits.dtype.type](x.ptr, b.ptr if b else None, ids.ptr, weights.ptr, tokens, experts, top, stream,
                             score=score, **more)
    stream.synchronize()
    i, w = ids.download(np.int32), weights.download(np.float32)
    assert (i[tokens * top:] == 77).all() and (w[tokens * top:] == 77).all()
    return i[: tokens * top].reshape(tokens, top), w[: tokens * top].reshape(tokens, top)


def check_route(stream, logits, bias, top, score, groups=1, top_groups=1, best=2, renormalize=True, scale=1.0):
    ids, weights = route(stream, logits, bias, top, score, groups=groups, top_groups=top_groups, group_best=best,
                         renormalize=renormalize, scale=scale)
    want_ids, want = mx.route(logits, bias, top, score, groups, top_groups, best, renormalize, scale)
    np.testing.assert_array_equal(ids, want_ids)
    # 64 bits throughout and one rounding to 32
    assert (np.abs(weights - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -148 + 1e-12 * np.abs(want)).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("score", [ops.SOFTMAX, ops.SIGMOID])
@pytest.mark.parametrize("tokens,experts,top", [(1, 1, 1), (1, 128, 8), (3, 8, 8), (5, 60, 6), (67, 64, 1), (130, 65, 4),
                                                (9, 160, 6), (33, 256, 8), (6, 300, 64), (4, 1024, 10), (3, 777, 3)])
def test_route(stream, tokens, experts, top, score, dtype):
    rng = np.random.default_rng(tokens + experts + top)
    logits = (rng.standard_normal((tokens, experts)) * 2).astype(dtype)
    check_route(stream, logits, None, top, score)
    bias = (rng.standard_normal(experts) * 0.1).astype(np.float32)
    check_route(stream, logits, bias, top, score, renormalize=False, scale=2.5)


@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("score", [ops.SOFTMAX, ops.SIGMOID])
@pytest.mark.parametrize("experts,groups,top_groups,top", [(8, 4, 1, 2), (8, 8, 3, 3), (60, 6, 2, 5), (64, 64, 9, 9),
                                                           (160, 8, 3, 6), (256, 8, 4, 8), (256, 2, 1, 8),
                                                           (256, 128, 5, 8), (1024, 16, 7, 12), (1024, 512, 11, 20),
                                                           (96, 3, 2, 40)])
def test_groups(stream, experts, groups, top_groups, top, score, best):
    rng = np.random.default_rng(experts + groups)
    logits = (rng.standard_normal((21, experts)) * 2).astype(np.float32)
    bias = (rng.standard_normal(experts) * 0.2).astype(np.float32)
    check_route(stream, logits, bias, top, score, groups, top_groups, best)
    check_route(stream, logits, None, top, score, groups, top_groups, best, renormalize=False)


@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
@pytest.mark.parametrize("score", [ops.SOFTMAX, ops.SIGMOID])
def test_masks_and_ties(stream, score, groups, top_groups):
    """Rows and groups that a mask leaves little or nothing of, the lowest value of the type in
    place of infinity, infinities and NaN, equal logits in lanes and slots alike."""
    experts, top = 160, 6
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((16, experts)).astype(np.float16)
    logits[0] = -np.inf
    logits[1, 1:] = -np.inf
    logits[2, : experts // 2] = -np.inf
    logits[3] = -65504
    logits[4, 4:] = -65504
    logits[5, ::3], logits[5, 1::3] = np.nan, np.inf
    logits[6] = np.nan
    logits[7] = 0.25
    logits[8] = np.round(logits[8])
    logits[9, 70:] = logits[9, 69]
    logits[10] = np.where(np.arange(experts) % 64 < 3, 1.0, -1.0)
    logits[11] = 65504
    logits[12, : experts // 4] = -np.inf
    logits[12, experts // 4 + 1: experts // 2] = -np.inf
    for dtype in (np.float16, np.float32):
        x = logits.astype(dtype)
        if dtype == np.float32:
            x[3], x[4, 4:] = np.finfo(np.float32).min, np.finfo(np.float32).min
        check_route(stream, x, None, top, score, groups, top_groups)
        bias = np.zeros(experts, np.float32)
        bias[5], bias[9], bias[11] = -np.inf, np.nan, np.inf
        bias[20:30] = -2.0  # choices below zero
        check_route(stream, x, bias, top, score, groups, top_groups)


def test_scores_that_32_bits_round_alike(stream):
    """Scores next to one another: 1 + 2^-24 apart, told apart."""
    logits = np.zeros((2, 64), np.float32)
    logits[0] = 8 + np.arange(64) * np.float32(2.0 ** -20)
    logits[1] = -logits[0]
    check_route(stream, logits, None, 5, ops.SIGMOID)
    check_route(stream, logits, np.zeros(64), 5, ops.SOFTMAX)


def plan(stream, ids, experts):
    tokens, top = ids.shape
    buffers = (DeviceBuffer.from_array(ids), DeviceBuffer.from_array(np.full(experts + 9, 55, np.int32)),
               DeviceBuffer.from_array(np.full(ids.size + 8, 55, np.int32)))
    ops.plan_experts(*[b.ptr for b in buffers], tokens, top, experts, stream)
    stream.synchronize()
    offsets, rows = buffers[1].download(np.int32), buffers[2].download(np.int32)
    assert (offsets[experts + 1:] == 55).all() and (rows[ids.size:] == 55).all()
    return offsets[: experts + 1], rows[: ids.size]


@pytest.mark.parametrize("tokens,top,experts", [(0, 4, 8), (1, 1, 1), (1, 8, 128), (2, 3, 5), (64, 4, 32), (65, 4, 1024),
                                                (1023, 1, 7), (1025, 4, 16), (4096, 8, 256), (8192, 4, 3),
                                                (5000, 7, 60), (20000, 8, 10)])
def test_plan(stream, tokens, top, experts):
    rng = np.random.default_rng(tokens + top)
    ids = rng.integers(-1, experts, (tokens, top)).astype(np.int32)
    want = mx.plan(ids, experts)
    for got, right in zip(plan(stream, ids, experts), want):
        np.testing.assert_array_equal(got, right)


def test_plan_of_strange_ids(stream):
    """None, the same expert twice, numbers that are no expert's, and all of one."""
    none = np.full((100, 4), -1, np.int32)
    strange = np.tile(np.array([[3, 3, 1 << 30, -(1 << 31)], [4, 1024, 2000, 0]], np.int32), (400, 1))
    one = np.full((3000, 2), 4, np.int32)
    for ids in (none, strange, one):
        for got, right in zip(plan(stream, ids, 5), mx.plan(np.where(ids < 5, ids, -1), 5)):
            np.testing.assert_array_equal(got, right)


def choices(rng, tokens, top, experts, holes=0.2, skew=1.0):
    """Distinct experts of each token, some tokens without."""
    liked = rng.standard_normal(experts) * skew
    ids = np.argsort(-(rng.gumbel(size=(tokens, experts)) + liked), axis=1)[:, :top].astype(np.int32)
    ids[rng.random(tokens) < holes] = -1
    return ids


class Case:
    """Weights, ids and the plan, on the host and on the device."""

    def __init__(self, rng, tokens, top, experts, hidden, inner, ids=None):
        self.sizes = tokens, top, experts, hidden, inner
        self.ids = choices(rng, tokens, top, experts) if ids is None else ids
        self.offsets, self.rows = mx.plan(self.ids, experts)
        self.up = mx.random_rows(rng, experts * 2 * inner, hidden, 4, 126, 129)
        self.back = mx.random_rows(rng, experts * hidden, inner, 4, 126, 129)
        self.weights = rng.standard_normal((tokens, top)).astype(np.float32)
        self.held = {k: DeviceBuffer.from_array(v) for k, v in
                     dict(ids=self.ids, offsets=self.offsets, rows=self.rows, up=self.up[0], up_s=self.up[1],
                          back=self.back[0], back_s=self.back[1], weights=self.weights).items()}

    def __getattr__(self, name):
        return self.__dict__["held"][name[:-4]].ptr if name.endswith("_ptr") else super().__getattribute__(name)

    def gate_up(self, stream, x, bits, small=1.0):
        tokens, top, experts, hidden, inner = self.sizes
        pairs = tokens * top
        xb = [DeviceBuffer.from_array(a) for a in x]
        h = DeviceBuffer.from_array(np.full(pairs * inner + 16, 0x7B7B, np.uint16))
        ops.experts_gate_up_silu_mx_f16(xb[0].ptr, xb[1].ptr, self.up_ptr, self.up_s_ptr, self.offsets_ptr,
                                        self.rows_ptr, h.ptr, tokens, top, experts, hidden, inner, bits, stream)
        stream.synchronize()
        raw = h.download(np.uint16)
        used = self.offsets[-1]
        assert (raw[used * inner:] == 0x7B7B).all(), "rows that no expert has are left alone"
        return raw[: used * inner].view(np.float16).reshape(used, inner)

    def check_gate_up(self, stream, rng, bits, low=121, high=124):
        tokens, top, experts, hidden, inner = self.sizes
        x = mx.random_rows(rng, tokens, hidden, bits, low, high)
        got = self.gate_up(stream, x, bits).astype(np.float64)
        w = mx.read(*self.up, 4).reshape(experts, 2 * inner, mx.padded(hidden))
        want, gate, up = mx.gate_up(mx.read(*x, bits), w, self.offsets, self.rows, top)
        assert np.abs(gate).max(initial=0) < 600 and np.abs(want).max(initial=0) < 65504
        assert (np.abs(got - want) <= (2.0 ** -11 + 2.0 ** -15) * np.abs(want) + 2.0 ** -25).all()

    def check_down(self, stream, rng, bits):
        tokens, top, experts, hidden, inner = self.sizes
        h = mx.random_rows(rng, max(tokens * top, 1), inner, bits, 120, 123)
        hb = [DeviceBuffer.from_array(a) for a in h]
        need = ops.experts_down_workspace(*self.sizes)
        work = DeviceBuffer.from_array(np.full(need + 64, 0xFF, np.uint8))  # NaN wherever nothing is written
        y = DeviceBuffer.from_array(np.full(tokens * hidden + 16, 0x7B7B, np.uint16))
        ops.experts_down_mx_f16(hb[0].ptr, hb[1].ptr, self.back_ptr, self.back_s_ptr, self.ids_ptr, self.offsets_ptr,
                                self.rows_ptr, self.weights_ptr, y.ptr, *self.sizes, bits, work.ptr, need, stream)
        stream.synchronize()
        assert (work.download(np.uint8)[need:] == 0xFF).all()
        raw = y.download(np.uint16)
        assert (raw[tokens * hidden:] == 0x7B7B).all()
        got = raw[: tokens * hidden].view(np.float16).reshape(tokens, hidden).astype(np.float64)
        w = mx.read(*self.back, 4).reshape(experts, hidden, mx.padded(inner))
        want, size = mx.down(mx.read(*h, bits), w, self.ids, self.offsets, self.rows, self.weights.astype(np.float64))
        assert size.max(initial=0) < 65504
        assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + (top + 1) * 2.0 ** -23 * size + 2.0 ** -25).all()
        assert (got[(self.ids < 0).all(1)] == 0).all()


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("tokens,top,experts,hidden,inner", [
    (1, 1, 1, 32, 32), (1, 8, 128, 256, 64), (3, 2, 8, 96, 160), (17, 4, 16, 416, 96), (64, 4, 32, 288, 32),
    (40, 2, 3, 160, 320), (150, 2, 4, 512, 96),        # tiles of 64 rows
    (700, 3, 9, 544, 160), (600, 2, 4, 640, 416),      # of 128 rows
    (2000, 2, 6, 512, 1600), (1030, 1, 2, 896, 6176),  # of 256 rows, for one of the two products at least
    (5, 3, 700, 64, 32), (30, 1, 1024, 128, 32)])
def test_products(stream, tokens, top, experts, hidden, inner, bits):
    rng = np.random.default_rng(tokens + experts + hidden + bits)
    case = Case(rng, tokens, top, experts, hidden, inner)
    case.check_gate_up(stream, rng, bits)
    case.check_down(stream, rng, bits)


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("tokens,top,experts,hidden,inner", [
    (60, 2, 8, 544, 416), (47, 4, 20, 1024, 160), (95, 1, 4, 512, 128), (96, 1, 4, 640, 96),  # 8 to 24 rows an expert
    (30, 8, 60, 1120, 512)])                                                          # few, in many tiles
def test_products_of_few_rows_each(stream, tokens, top, experts, hidden, inner, bits):
    rng = np.random.default_rng(tokens + experts + hidden + bits)
    case = Case(rng, tokens, top, experts, hidden, inner)
    case.check_gate_up(stream, rng, bits)
    case.check_down(stream, rng, bits)


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("tokens,experts", [(150, 3), (190, 3), (130, 20), (700, 2), (1100, 3)])
def test_one_expert_of_several_tiles(stream, tokens, experts, bits):
    """More rows of one expert than the mean, by which the tiles are chosen, lets expect."""
    rng = np.random.default_rng(tokens + bits)
    ids = np.where(rng.random((tokens, 1)) < 0.95, 1, rng.integers(-1, experts, (tokens, 1))).astype(np.int32)
    case = Case(rng, tokens, 1, experts, 544, 672, ids)
    case.check_gate_up(stream, rng, bits)
    case.check_down(stream, rng, bits)


@pytest.mark.parametrize("hidden,inner", [(8192, 64), (8224, 32), (64, 8192), (32, 16384), (32, 16416)])
def test_long_rows_of_few_tokens(stream, hidden, inner):
    rng = np.random.default_rng(hidden + inner)
    case = Case(rng, 5, 2, 3, hidden, inner)
    case.check_gate_up(stream, rng, 4, 118, 121)
    case.check_down(stream, rng, 6)


@pytest.mark.parametrize("tokens", [3, 200])
@pytest.mark.parametrize("which", ["none", "one", "twice", "last"])
def test_uneven_choices(stream, which, tokens):
    """No token has an expert; all have one; each the same one twice; only the last expert is used."""
    rng = np.random.default_rng(tokens)
    ids = {"none": np.full((tokens, 2), -1), "one": np.tile([[1, -1]], (tokens, 1)),
           "twice": np.full((tokens, 2), 3), "last": np.tile([[-1, 6]], (tokens, 1))}[which].astype(np.int32)
    case = Case(rng, tokens, 2, 7, 160, 96, ids)
    case.check_gate_up(stream, rng, 6)
    case.check_down(stream, rng, 6)


def test_no_inner_or_hidden_elements(stream):
    """Nothing to add up is zero."""
    rng = np.random.default_rng(0)
    case = Case(rng, 5, 2, 4, 64, 0)
    case.check_down(stream, rng, 4)
    case = Case(rng, 5, 2, 4, 0, 64)
    got = case.gate_up(stream, mx.random_rows(rng, 5, 0, 4), 4)
    assert (got == 0).all()


def test_offsets_past_the_rows(stream):
    """A plan that does not fit is cut to the pairs there are: nothing outside is written."""
    rng = np.random.default_rng(4)
    tokens, top, experts, hidden, inner = 6, 2, 4, 64, 32
    case = Case(rng, tokens, top, experts, hidden, inner, choices(rng, tokens, top, experts, 0.0))
    x = [DeviceBuffer.from_array(a) for a in mx.random_rows(rng, tokens, hidden, 4)]
    h = DeviceBuffer.from_array(np.full(tokens * top * inner + 64, 0x7B7B, np.uint16))
    for offsets in ([0, 100, 1 << 30, 5, 2000], [-5, -1, 3, 3, 13], [9, 2, 50, 1, 12]):
        for rows in (case.rows, np.full(12, -1), np.full(12, 1 << 30)):
            o = DeviceBuffer.from_array(np.array(offsets, np.int32))
            r = DeviceBuffer.from_array(rows.astype(np.int32))
            ops.experts_gate_up_silu_mx_f16(x[0].ptr, x[1].ptr, case.up_ptr, case.up_s_ptr, o.ptr, r.ptr, h.ptr, tokens,
                                            top, experts, hidden, inner, 4, stream)
            stream.synchronize()
            assert (h.download(np.uint16)[tokens * top * inner:] == 0x7B7B).all()


def test_last_of_many_experts(stream):
    """Weights of more than 4 GB: the last expert's."""
    rng = np.random.default_rng(8)
    experts, hidden, inner = 1024, 4096, 1056
    up = mx.random_rows(rng, 2 * inner, hidden, 4, 126, 129)
    each, each_s = up[0].nbytes, up[1].nbytes
    assert experts * each > 1 << 32
    values, scales = DeviceBuffer(experts * each), DeviceBuffer(experts * each_s)
    values.upload(up[0], offset=(experts - 1) * each)
    scales.upload(up[1], offset=(experts - 1) * each_s)
    for tokens in (3, 9000):
        ids = np.full((tokens, 1), experts - 1, np.int32)
        offsets, rows = mx.plan(ids[:50], experts)
        offsets[-1] = tokens
        rows = np.arange(tokens, dtype=np.int32)
        x = mx.random_rows(rng, tokens, hidden, 6, 117, 120)
        b = [DeviceBuffer.from_array(a) for a in (*x, offsets, rows)]
        h = DeviceBuffer(tokens * inner * 2)
        ops.experts_gate_up_silu_mx_f16(b[0].ptr, b[1].ptr, values.ptr, scales.ptr, b[2].ptr, b[3].ptr, h.ptr, tokens, 1,
                                        experts, hidden, inner, 6, stream)
        stream.synchronize()
        n = 3
        got = h.download(np.float16, count=n * inner, offset=(tokens - n) * inner * 2).reshape(n, inner)
        xv = mx.read(x[0][-n:], x[1][-n:], 6)
        want, _, _ = mx.gate_up(xv, mx.read(*up, 4)[None], np.array([0, n]), np.arange(n), 1)
        assert (np.abs(got - want) <= (2.0 ** -11 + 2.0 ** -15) * np.abs(want) + 2.0 ** -25).all()
    values.free()
    scales.free()


@pytest.mark.parametrize("tokens", [4, 300])
def test_captured_and_replayed(stream, tokens):
    """From logits to output in one captured graph, replayed as the logits and activations
    change, each replay equal to the same calls made at once."""
    top, experts, hidden, inner = 3, 16, 256, 160
    rng = np.random.default_rng(tokens)
    case = Case(rng, tokens, top, experts, hidden, inner)
    pairs = tokens * top
    room = {k: DeviceBuffer(n) for k, n in dict(
        logits=tokens * experts * 4, x=tokens * hidden * 2, ids=pairs * 4, weights=pairs * 4, offsets=(experts + 1) * 4,
        rows=pairs * 4, xv=tokens * ops.mx_value_bytes(hidden, 6), xs=tokens * ops.mx_scale_bytes(hidden),
        h=pairs * inner * 2, hv=pairs * ops.mx_value_bytes(inner, 6), hs=pairs * ops.mx_scale_bytes(inner),
        y=tokens * hidden * 2, work=ops.experts_down_workspace(tokens, top, experts, hidden, inner)).items()}
    p = {k: b.ptr for k, b in room.items()}
    room["h"].upload(np.zeros(pairs * inner, np.float16))  # rows that no expert has are quantised too

    def calls(s):
        ops.route_experts_f32(p["logits"], None, p["ids"], p["weights"], tokens, experts, top, s)
        ops.plan_experts(p["ids"], p["offsets"], p["rows"], tokens, top, experts, s)
        ops.mx_quantize_f16(p["x"], p["xv"], p["xs"], tokens, hidden, 6, s)
        ops.experts_gate_up_silu_mx_f16(p["xv"], p["xs"], case.up_ptr, case.up_s_ptr, p["offsets"], p["rows"], p["h"],
                                        tokens, top, experts, hidden, inner, 6, s)
        ops.mx_quantize_f16(p["h"], p["hv"], p["hs"], pairs, inner, 6, s)
        ops.experts_down_mx_f16(p["hv"], p["hs"], case.back_ptr, case.back_s_ptr, p["ids"], p["offsets"], p["rows"],
                                p["weights"], p["y"], tokens, top, experts, hidden, inner, 6, p["work"],
                                room["work"].nbytes, s)

    def fill():
        logits = rng.standard_normal((tokens, experts)).astype(np.float32)
        logits[rng.random(tokens) < 0.2] = -np.inf
        room["logits"].upload(logits)
        room["x"].upload((rng.standard_normal((tokens, hidden)) * 0.05).astype(np.float16))

    rt = HipRuntime()
    fill()
    calls(stream)
    stream.synchronize()
    graph = rt.capture(stream, lambda: calls(stream))
    for _ in range(4):
        fill()
        calls(stream)
        stream.synchronize()
        want = room["y"].download(np.uint16)
        room["y"].upload(np.full(tokens * hidden, 0x7B7B, np.uint16))
        rt.launch_graph(graph, stream)
        stream.synchronize()
        np.testing.assert_array_equal(room["y"].download(np.uint16), want)
    rt.destroy_graph(graph)
