"""Products of microscaled rows against 64 bits.

Most inputs are such that 32-bit sums are exact: with scales 2^-1, 1 and 2 on each side
products are multiples of 2^-4 2^-2 and below 2^6 2^2; a sum that stays under 2^18 then fits 24
bits in any order, and 4096 or more random terms of a mean square under 2^10 stay far under
that.  Such outputs have to be equal, the f16 ones to the rounded sum."""

from __future__ import annotations

import numpy as np
import pytest

import mx_oracle as mx
from mote_amd import ops
from mote_amd.device import DeviceBuffer, Stream

pytestmark = pytest.mark.gpu


def linear(stream, x, w, rows, n, k, bits, f16=True, fill=0x7B7B):
    buffers = [DeviceBuffer.from_array(a) for a in (*x, *w)]
    dtype = np.float16 if f16 else np.float32
    y = DeviceBuffer.from_array(np.full(rows * n * dtype().itemsize // 2 + 32, fill, np.uint16))
    (ops.mx_linear_f16 if f16 else ops.mx_linear_f32)(*[b.ptr for b in buffers], y.ptr, rows, n, k, bits, stream)
    stream.synchronize()
    raw = y.download(np.uint16)
    assert (raw[-32:] == fill).all(), "written past the output"
    return raw[:-32].view(dtype).reshape(rows, n)


def exact(x, w, bits):
    return mx.read(*x, bits) @ mx.read(*w, 4).T


def check(stream, rows, n, k, bits, f16, seed=0):
    rng = np.random.default_rng(seed + rows * 31 + n * 7 + k)
    x, w = mx.random_rows(rng, rows, k, bits, 126, 129), mx.random_rows(rng, n, k, 4, 126, 129)
    got = linear(stream, x, w, rows, n, k, bits, f16)
    want = exact(x, w, bits)
    assert np.abs(want).max() < 2 ** 15
    np.testing.assert_array_equal(got, want.astype(got.dtype))


# rows on each side of every tile's and rule's borders, columns and K that fill none
@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 32, 33, 48, 64, 65, 100, 129, 257])
@pytest.mark.parametrize("n,k", [(1, 32), (17, 96), (64, 128), (33, 416), (16, 512), (130, 2880), (1000, 1120)])
def test_linear(stream, rows, n, k, bits):
    check(stream, rows, n, k, bits, (rows + n) % 2 == 0)


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("rows,n,k", [
    (1, 14336, 4096), (16, 4097, 4096),      # columns in twos and more of a workgroup
    (1, 300, 8192), (5, 300, 8320), (16, 100, 16384), (3, 100, 16416),  # K at the waves' and kernels' limits
    (200, 2050, 640), (400, 1027, 544),      # tiles of 64 x 64 and 32 x 64
    (500, 3001, 672), (1100, 2100, 512),     # of 128 x 64 and 128 x 128
    (3500, 3600, 544), (3400, 3700, 896), (3333, 3585, 1024),  # of 256 x 256, 5, 7 and 8 steps
])
def test_larger(stream, rows, n, k, bits):
    check(stream, rows, n, k, bits, rows % 2 == 0)


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("rows,n,k", [
    (1, 12225, 512), (7, 12289, 2880), (32, 12300, 416), (31, 12777, 640),  # 64 x 32, K in two
    (100, 3100, 1184), (200, 1790, 544), (257, 1400, 896), (33, 6111, 800),
    (17, 200, 8320), (16, 6100, 8224), (16, 6113, 8224), (2, 64, 65536),    # long rows, few and more of them
])
def test_few_rows(stream, rows, n, k, bits):
    check(stream, rows, n, k, bits, rows % 2 == 0)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_no_features_and_nothing(stream, rows):
    empty = np.zeros(16, np.uint8)
    got = linear(stream, (empty, empty), (empty, empty), rows, 50, 0, 4)
    assert (got == 0).all()
    y = DeviceBuffer.from_array(np.full(8, 7, np.uint16))
    w = DeviceBuffer.from_array(empty)
    ops.mx_linear_f16(w.ptr, w.ptr, w.ptr, w.ptr, y.ptr, 0, 8, 32, 4, stream)
    ops.mx_linear_f16(w.ptr, w.ptr, w.ptr, w.ptr, y.ptr, 8, 0, 32, 4, stream)
    stream.synchronize()
    assert (y.download(np.uint16) == 7).all()


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("rows,n,k", [(3, 50, 1024), (40, 64, 1024), (300, 520, 1024)])
def test_wide_scales(stream, rows, n, k, bits):
    """Scales 2^-20 to 2^19 on both sides.  A step's four blocks and the sum before
    meet in an addition of 32 bits each, rounded or cut: K / 32 + K / 128 of them, each off by
    less than 2^-23 of the largest partial sum, which the sum of all sizes bounds."""
    rng = np.random.default_rng(rows)
    x, w = mx.random_rows(rng, rows, k, bits, 107, 147), mx.random_rows(rng, n, k, 4, 107, 147)
    got = linear(stream, x, w, rows, n, k, bits, False)
    xv, wv = mx.read(*x, bits), mx.read(*w, 4)
    bound = (k / 32 + k / 128) * 2.0 ** -23 * (np.abs(xv) @ np.abs(wv).T)
    assert (np.abs(got - xv @ wv.T) <= bound).all()


@pytest.mark.parametrize("rows,n", [(2, 40), (20, 40), (70, 200), (600, 2000)])
def test_not_a_number(stream, rows, n):
    """A scale of 255 shows in its row's outputs, zeros beside it or not, and nowhere else."""
    k, rng = 640, np.random.default_rng(n)
    x, w = mx.random_rows(rng, rows, k, 6, 126, 129), mx.random_rows(rng, n, k, 4, 126, 129)
    x[1][1, 7] = 255
    w[1][n - 3, 19] = 255
    x[0][rows - 1] = 0
    got = linear(stream, x, w, rows, n, k, 6, False)
    bad = np.zeros((rows, n), bool)
    bad[1], bad[:, n - 3] = True, True
    assert np.isnan(got[bad]).all()
    x[1][1, 7] = w[1][n - 3, 19] = 127
    np.testing.assert_array_equal(got[~bad], exact(x, w, 6)[~bad])


@pytest.mark.parametrize("rows", [4, 30, 500])
def test_padding_may_hold_any_scale_but_nan(stream, rows):
    """Values of the padding are zeros: its scales do not matter."""
    n, k, rng = 70, 160, np.random.default_rng(rows)
    x, w = mx.random_rows(rng, rows, k, 4, 126, 129), mx.random_rows(rng, n, k, 4, 126, 129)
    want = exact(x, w, 4)
    x[1][:, 5:], w[1][:, 5:] = 140, 150
    np.testing.assert_array_equal(linear(stream, x, w, rows, n, k, 4, False), want)


def test_weights_past_32_bits(stream):
    """The last outputs of weights of more than 4 GB."""
    n, k = (1 << 32) // 2048 + 300, 4096
    rng = np.random.default_rng(5)
    last = 40
    w = mx.random_rows(rng, last, k, 4, 126, 129)
    values, scales = DeviceBuffer(n * k // 2), DeviceBuffer(n * k // 32)
    values.upload(w[0], offset=(n - last) * k // 2)
    scales.upload(w[1], offset=(n - last) * k // 32)
    for rows in (1, 40):
        x = mx.random_rows(rng, rows, k, 6, 126, 129)
        xb = [DeviceBuffer.from_array(a) for a in x]
        y = DeviceBuffer(rows * n * 4)
        ops.mx_linear_f32(xb[0].ptr, xb[1].ptr, values.ptr, scales.ptr, y.ptr, rows, n, k, 6, stream)
        stream.synchronize()
        want = exact(x, w, 6)
        for r in range(rows):
            got = y.download(np.float32, count=last, offset=(r * n + n - last) * 4)
            np.testing.assert_array_equal(got, want[r])
        y.free()
    values.free()
    scales.free()


def test_two_streams_at_once(stream):
    """Calls on two streams, without waiting between: nothing is shared."""
    rng, other = np.random.default_rng(9), Stream()
    held = []
    for s, rows in ((stream, 3), (other, 40), (stream, 300), (other, 7)):
        x, w = mx.random_rows(rng, rows, 1024, 4, 126, 129), mx.random_rows(rng, 500, 1024, 4, 126, 129)
        buffers = [DeviceBuffer.from_array(a) for a in (*x, *w)]
        y = DeviceBuffer(rows * 500 * 4)
        held.append((s, rows, buffers, y, exact(x, w, 4)))
    for s, rows, buffers, y, _ in held:
        ops.mx_linear_f32(*[b.ptr for b in buffers], y.ptr, rows, 500, 1024, 4, s)
    stream.synchronize()
    other.synchronize()
    for _, rows, _, y, want in held:
        np.testing.assert_array_equal(y.download(np.float32).reshape(rows, 500), want)
    other.close()
