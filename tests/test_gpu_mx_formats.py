"""Rows to microscaled 4 and 6 bits and back, code for code against the oracle."""

from __future__ import annotations

import numpy as np
import pytest

import mx_oracle as mx
from mote_amd import ops
from mote_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu

TYPES = {"f16": (np.float16, ops.mx_quantize_f16, ops.mx_dequantize_f16),
         "f32": (np.float32, ops.mx_quantize_f32, ops.mx_dequantize_f32)}


def quantize(stream, x, bits, type, stride=None, skip=0):
    dtype, fn, _ = TYPES[type]
    rows, features = x.shape
    s = stride or features
    flat = np.full(skip + rows * s, np.nan, dtype)  # between the rows: never read
    flat[skip:].reshape(rows, s)[:, :features] = x
    source = DeviceBuffer.from_array(flat)
    values = DeviceBuffer.from_array(np.full(rows * ops.mx_value_bytes(features, bits) + 32, 0xA5, np.uint8))
    scales = DeviceBuffer.from_array(np.full(rows * ops.mx_scale_bytes(features) + 32, 0xA5, np.uint8))
    fn(source.ptr + skip * flat.itemsize, values.ptr, scales.ptr, rows, features, bits, stream, stride=stride)
    stream.synchronize()
    v, s = values.download(np.uint8), scales.download(np.uint8)
    assert (v[-32:] == 0xA5).all() and (s[-32:] == 0xA5).all()
    return v[:-32].reshape(rows, -1), s[:-32].reshape(rows, -1)


def same_codes(got, want, bits):
    """The same values and scales; a zero may have either sign."""
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(mx.elements(bits)[mx.unpack(got[0], bits)], mx.elements(bits)[mx.unpack(want[0], bits)])


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("rows,features", [(1, 32), (1, 4096), (3, 96), (5, 160), (7, 2880), (300, 64), (65, 8192)])
def test_quantize(stream, rows, features, bits, type):
    rng = np.random.default_rng(rows + features + bits)
    x = (rng.standard_normal((rows, features)) * 2.0 ** rng.integers(-9, 9, (rows, 1))).astype(TYPES[type][0])
    got = quantize(stream, x, bits, type)
    same_codes(got, mx.quantize(x, bits), bits)
    width = features * bits // 8
    if features % 128:  # the padding
        blocks = features // 32
        assert (got[1][:, blocks:] == 0).all()
        assert (mx.unpack(got[0], bits)[:, features:] == 0).all() and width < got[0].shape[1]


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("skip,stride", [(0, 200), (1, 161), (3, 1000)])
def test_strides_and_odd_addresses(stream, bits, skip, stride):
    rng = np.random.default_rng(stride)
    for type in ("f16", "f32"):
        x = rng.standard_normal((9, 160)).astype(TYPES[type][0])
        same_codes(quantize(stream, x, bits, type, stride, skip), mx.quantize(x, bits), bits)


@pytest.mark.parametrize("bits", [4, 6])
def test_every_f16(stream, bits):
    """Each binary16 as a block's largest with each of a few others beside it."""
    every = np.arange(1 << 16, dtype=np.uint16).view(np.float16)
    every = every[np.isfinite(every)]
    x = np.zeros((every.size, 32), np.float16)
    x[:, 0] = every
    with np.errstate(under="ignore"):
        for i, part in enumerate((0.75, 0.6250, 0.5, -0.4375, 0.3125, -0.25, 0.171875, 0.125, 0.0625, 0.046875, 0.03125)):
            x[:, 1 + i] = every * np.float16(part)
    same_codes(quantize(stream, x, bits, "f16"), mx.quantize(x, bits), bits)


@pytest.mark.parametrize("bits", [4, 6])
def test_ties_and_limits_in_f32(stream, bits):
    """Halfway between elements and a step of 32 bits to each side, at scales
    from the smallest to the largest."""
    up = mx.UP[bits]
    middle = ((up[1:] + up[:-1]) / 2).astype(np.float32)
    near = np.concatenate([middle, np.nextafter(middle, np.float32(0)), np.nextafter(middle, np.float32(9))])
    near = np.concatenate([near, -near, [up[-1], 7.75, 7.9999995]]).astype(np.float32)
    near = np.concatenate([near, np.zeros(-near.size % 31, np.float32)]).reshape(-1, 31)
    rows = []
    for e in (-149, -140, -127, -126, -125, -124, -100, -96, -95, -60, -1, 0, 1, 90, 124, 125):
        top = np.full((len(near), 1), 4.0, np.float32)  # 4 to 7.99: exponent 2
        with np.errstate(under="ignore"):
            rows.append(np.ldexp(np.concatenate([top, near], 1), e).astype(np.float32))
    x = np.concatenate(rows)
    same_codes(quantize(stream, x, bits, "f32"), mx.quantize(x, bits), bits)


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("bits", [4, 6])
def test_not_finite(stream, bits, type):
    dtype, _, back = TYPES[type]
    x = np.ones((4, 96), dtype)
    x[0, 5], x[1, 40], x[2, 95] = np.nan, np.inf, -np.inf
    got = quantize(stream, x, bits, type)
    same_codes(got, mx.quantize(x, bits), bits)
    values, scales, out = (DeviceBuffer.from_array(got[0]), DeviceBuffer.from_array(got[1]),
                           DeviceBuffer(4 * 96 * dtype().itemsize))
    back(values.ptr, scales.ptr, out.ptr, 4, 96, bits, stream)
    stream.synchronize()
    y = out.download(dtype).reshape(4, 3, 32)
    bad = np.zeros((4, 3), bool)
    bad[0, 0] = bad[1, 1] = bad[2, 2] = True
    assert np.isnan(y[bad]).all() and (y[~bad] == 1).all()


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("features,stride", [(96, None), (2048, None), (160, 171)])
def test_dequantize_every_scale(stream, features, stride, bits, type):
    """Random codes at every scale byte; what lies between the rows is kept."""
    dtype, _, back = TYPES[type]
    rng = np.random.default_rng(features)
    values, scales = mx.random_rows(rng, 256, features, bits)
    scales[:, : features // 32] = np.arange(256)[:, None]
    s = stride or features
    mark = dtype(123)
    out = DeviceBuffer.from_array(np.full(256 * s, mark, dtype))
    buffers = DeviceBuffer.from_array(values), DeviceBuffer.from_array(scales)
    back(buffers[0].ptr, buffers[1].ptr, out.ptr, 256, features, bits, stream, stride=stride)
    stream.synchronize()
    got = out.download(dtype).reshape(256, s)
    with np.errstate(over="ignore", under="ignore"):
        want = mx.read(values, scales, bits)[:, :features].astype(dtype)
    np.testing.assert_array_equal(got[:, :features], want)
    assert (got[:, features:] == mark).all()


def test_rows_past_32_bits(stream):
    """The last of rows whose elements pass 2^32: its address is right."""
    rows, features = (1 << 32) // 8192 + 3, 8192
    x = np.random.default_rng(1).standard_normal((1, features)).astype(np.float16)
    source = DeviceBuffer(rows * features * 2)
    source.upload(x, offset=(rows - 1) * features * 2)
    values, scales = DeviceBuffer(rows * features // 2), DeviceBuffer(rows * features // 32)
    ops.mx_quantize_f16(source.ptr, values.ptr, scales.ptr, rows, features, 4, stream)
    stream.synchronize()
    got = (values.download(np.uint8, offset=(rows - 1) * features // 2)[None],
           scales.download(np.uint8, offset=(rows - 1) * features // 32)[None])
    same_codes(got, mx.quantize(x, 4), 4)
    ops.mx_dequantize_f16(values.ptr, scales.ptr, source.ptr, rows, features, 4, stream)
    stream.synchronize()
    back = source.download(np.float16, offset=(rows - 1) * features * 2)
    np.testing.assert_array_equal(back, mx.read(*got, 4)[0].astype(np.float16))
    for b in (source, values, scales):
        b.free()
