"""The experts' MLP from logits to output as a layer runs it: each step of ExpertsMX
against the oracle on what the step before gave, and the example."""

from __future__ import annotations

import os
import sys

import numpy as np
import pytest

import mx_oracle as mx
from mote_amd import ops
from mote_amd.device import DeviceBuffer
from mote_amd.experts import ExpertsMX
from mote_amd.hip_runtime import HipRuntime

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("bits,logits_f16", [(4, False), (6, True)])
@pytest.mark.parametrize("tokens,top,experts,hidden,inner",
                         [(1, 2, 4, 64, 32), (37, 3, 8, 288, 160), (260, 2, 4, 544, 96)])
def test_steps(stream, tokens, top, experts, hidden, inner, bits, logits_f16):
    rng = np.random.default_rng(tokens + bits)
    bias = 0.1 * rng.standard_normal(experts)
    block = ExpertsMX(experts, top, hidden, inner, 300, bits, score=ops.SIGMOID, bias=bias, scale=1.5)
    weights = [[rng.standard_normal(s).astype(np.float32) / np.sqrt(s[1])
                for s in ((inner, hidden), (inner, hidden), (hidden, inner))] for _ in range(experts)]
    for e, w in enumerate(weights):
        block.load(e, *w, stream)
    stride = hidden + 24
    x = np.zeros((tokens, stride), np.float16)
    x[:, :hidden] = rng.standard_normal((tokens, hidden))
    logits = rng.standard_normal((tokens, experts)).astype(np.float16 if logits_f16 else np.float32)
    logits[tokens // 2:][:2] = -np.inf if tokens > 1 else 0
    held = DeviceBuffer.from_array(x), DeviceBuffer.from_array(logits)
    y = DeviceBuffer(tokens * hidden * 2)
    block.forward(held[0].ptr, held[1].ptr, y.ptr, tokens, stream, logits_f16=logits_f16, stride=stride)
    stream.synchronize()

    want_ids, want_weights = mx.route(logits, np.asarray(bias, np.float32), top, ops.SIGMOID, scale=1.5)
    ids = block.ids.download(np.int32, count=tokens * top).reshape(tokens, top)
    np.testing.assert_array_equal(ids, want_ids)
    offsets, rows = mx.plan(ids, experts)
    used = offsets[-1]
    # gate and up: weights and x rounded by the oracle; silu and one rounding, products of
    # x's and the weights' elements in 32 bits, each of the K / 32 + K / 128 sums good to 2^-23 of
    # the sizes' sum, which the other factor (up to 1 + |gate| in silu's slope) carries on
    xv = mx.read(*mx.quantize(x[:, :hidden], bits), bits)
    up = np.stack([np.concatenate([mx.read(*mx.quantize(w[i], 4), 4) for i in (0, 1)]) for w in weights])
    want, gate, lift = mx.gate_up(xv, up, offsets, rows, top)
    size = np.zeros((used, 2 * inner))
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        size[a:b] = np.abs(xv[rows[a:b] // top]) @ np.abs(up[e]).T
    off = (hidden / 32 + hidden / 128 + 5) * 2.0 ** -23 * size
    bound = 1.1 * off[:, :inner] * np.abs(lift) + np.abs(gate) * off[:, inner:] + 2 * off[:, :inner] * off[:, inner:]
    h = block._h.download(np.float16, count=used * inner).reshape(used, inner)
    assert (np.abs(h - want) <= bound + (2.0 ** -11 + 2.0 ** -15) * np.abs(want) + 2.0 ** -25).all()
    # down: of the h there is
    hv = np.zeros((tokens * top, mx.padded(inner)))
    hv[:used] = mx.read(*mx.quantize(h, bits), bits)
    back = np.stack([mx.read(*mx.quantize(w[2], 4), 4) for w in weights])
    total, sizes = mx.down(hv, back, ids, offsets, rows, want_weights)
    deep = np.zeros((tokens, hidden))
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        for i in range(a, b):
            t, j = divmod(int(rows[i]), top)
            deep[t] += abs(want_weights[t, j]) * (np.abs(hv[i]) @ np.abs(back[e]).T)
    got = y.download(np.float16).reshape(tokens, hidden)
    bound = 2.0 ** -11 * np.abs(total) + (inner / 32 + inner / 128 + top + 4) * 2.0 ** -23 * deep + 2.0 ** -25
    assert (np.abs(got - total) <= bound).all()
    block.free()


def test_two_graphs(stream):
    """Calls of two sizes captured, replayed in turn with other inputs: each equal to the call made
    at once, though they share the object's memory."""
    tokens, top, experts, hidden, inner = (200, 3), 2, 8, 256, 96
    rng = np.random.default_rng(9)
    block = ExpertsMX(experts, top, hidden, inner, 200)
    for e in range(experts):
        block.load(e, *(rng.standard_normal(s).astype(np.float32) / np.sqrt(s[1])
                        for s in ((inner, hidden), (inner, hidden), (hidden, inner))), stream)
    x, logits, y = (DeviceBuffer(n) for n in (tokens[0] * hidden * 2, tokens[0] * experts * 4, tokens[0] * hidden * 2))
    rt = HipRuntime()
    graphs = [rt.capture(stream, lambda n=n: block.forward(x.ptr, logits.ptr, y.ptr, n, stream)) for n in tokens]
    for i in range(6):
        n = tokens[i % 2]
        x.upload(rng.standard_normal((tokens[0], hidden)).astype(np.float16))
        logits.upload(rng.standard_normal((tokens[0], experts)).astype(np.float32))
        block.forward(x.ptr, logits.ptr, y.ptr, n, stream)
        stream.synchronize()
        want = y.download(np.uint16, count=n * hidden)
        y.upload(np.full(tokens[0] * hidden, 0x7B7B, np.uint16))
        rt.launch_graph(graphs[i % 2], stream)
        stream.synchronize()
        np.testing.assert_array_equal(y.download(np.uint16, count=n * hidden), want)
        assert (y.download(np.uint16)[n * hidden:] == 0x7B7B).all()
    for graph in graphs:
        rt.destroy_graph(graph)
    block.free()


def test_refusals(stream):
    for bad in (dict(experts=0), dict(top=5), dict(top=0), dict(hidden=33), dict(inner=0), dict(max_tokens=0),
                dict(bits=8), dict(bias=np.zeros(3))):
        with pytest.raises(ValueError):
            ExpertsMX(**{**dict(experts=4, top=2, hidden=64, inner=32, max_tokens=8), **bad})
    block = ExpertsMX(4, 2, 64, 32, 8)
    w = np.zeros((32, 64), np.float32), np.zeros((32, 64), np.float32), np.zeros((64, 32), np.float32)
    with pytest.raises(ValueError):
        block.load(4, *w, stream)
    with pytest.raises(ValueError):
        block.load(0, w[0], w[1], w[0], stream)
    with pytest.raises(ValueError):
        block.forward(block._x.ptr, block._x.ptr, block._x.ptr, 9, stream)
    block.free()


def test_example(stream):
    """The example runs; tokens alone and together agree but for what their sums' order
    moves over a rounding (6 bits: a sixteenth of the element, in few of them)."""
    import decoder_experts

    together, alone = decoder_experts.run(hidden=256, inner=96, experts=8, top=2, tokens=40, single=3)
    assert np.isfinite(together).all() and np.isfinite(alone).all()
    assert np.abs(together - alone).max() <= 2.0 ** -4 * np.abs(together).max()
