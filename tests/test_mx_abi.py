"""What the microscaled formats' and the experts' entry points refuse, and the
calls that have nothing to do (CPU: every check comes before any device work, so
stand-in pointers are never followed); the oracle's own arithmetic."""

from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest

import mx_oracle as mx

FAKE = 0x10000
STREAM = 0x20000
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def lib():
    from mote_amd import _ffi

    if not os.path.exists(_ffi.LIBRARY):
        from mote_amd import build

        build.build()
    return _ffi.lib()


def refusals(fn, good, bad):
    for at, values in bad.items():
        for v in values:
            args = list(good)
            args[at] = v
            assert fn(*args) == -1, (at, v)


def nothing(fn, good, at):
    for i in at:
        args = list(good)
        args[i] = 0
        assert fn(*args) == 0, i


@pytest.mark.parametrize("name,size", [("quantize_f16", 2), ("quantize_f32", 4)])
def test_quantize(lib, name, size):
    fn = getattr(lib, "mote_hip_mx_" + name)
    good = [FAKE, FAKE, FAKE, 5, 96, 100, 4, STREAM]
    refusals(fn, good, {0: [None, FAKE + size // 2], 1: [None, FAKE + 8], 2: [None], 3: [(1 << 31) + 1, 1 << 63],
                        4: [95, (1 << 24) + 32, 1 << 40], 5: [95, 1 << 41], 6: [0, 5, 8, -4], 7: [None]})
    assert fn(FAKE, FAKE, FAKE, 1 << 31, 64, 64, 4, STREAM) == -1  # more blocks than one launch
    nothing(fn, good, [3, 4])


@pytest.mark.parametrize("name,size", [("dequantize_f16", 2), ("dequantize_f32", 4)])
def test_dequantize(lib, name, size):
    fn = getattr(lib, "mote_hip_mx_" + name)
    good = [FAKE, FAKE, FAKE, 5, 96, 100, 6, STREAM]
    refusals(fn, good, {0: [None, FAKE + 8], 1: [None], 2: [None, FAKE + size // 2], 3: [(1 << 31) + 1], 4: [95],
                        5: [95], 6: [0, 5, 8], 7: [None]})
    nothing(fn, good, [3, 4])


@pytest.mark.parametrize("name,size", [("f16", 2), ("f32", 4)])
def test_linear(lib, name, size):
    fn = getattr(lib, "mote_hip_mx_linear_" + name)
    good = [FAKE] * 5 + [7, 33, 96, 4, STREAM]
    refusals(fn, good, {0: [None, FAKE + 8], 1: [None, FAKE + 2], 2: [None, FAKE + 8], 3: [None, FAKE + 1],
                        4: [None, FAKE + size // 2], 5: [(1 << 30) + 1], 6: [(1 << 24) + 1], 7: [95, (1 << 24) + 32],
                        8: [0, 3, 8], 9: [None]})
    assert fn(*[FAKE] * 5, 1 << 30, 1 << 24, 512, 4, STREAM) == -1  # more work than one launch
    nothing(fn, good, [5, 6])


def test_route(lib):
    for name, size in (("f16", 2), ("f32", 4)):
        fn = getattr(lib, "mote_hip_route_experts_" + name)
        good = [FAKE, FAKE, FAKE, FAKE, 3, 64, 8, 0, 8, 4, 2, 1, 1.0, STREAM]
        refusals(fn, good, {0: [None, FAKE + size // 2], 1: [FAKE + 2], 2: [None, FAKE + 2], 3: [None, FAKE + 2],
                            4: [1 << 26, 1 << 31], 5: [1025, 60], 6: [65, 33], 7: [-1, 2], 8: [0, 7], 9: [0, 9],
                            10: [0, 3], 11: [-1, 2], 12: [NAN, INF], 13: [None]})
        nothing(fn, good, [4, 6])
        assert fn(FAKE, None, FAKE, FAKE, 3, 0, 0, 1, 1, 1, 1, 0, 1.0, STREAM) == 0
        assert fn(FAKE, None, FAKE, FAKE, 3, 4, 5, 1, 1, 1, 1, 0, 1.0, STREAM) == -1  # more than there are


def test_plan(lib):
    fn = lib.mote_hip_plan_experts
    good = [FAKE, FAKE, FAKE, 5, 4, 16, STREAM]
    refusals(fn, good, {0: [None, FAKE + 2], 1: [None, FAKE + 2], 2: [None, FAKE + 2], 3: [1 << 31, 1 << 29], 4: [65],
                        5: [1025], 6: [None]})
    nothing(fn, good, [5])


def test_gate_up(lib):
    fn = lib.mote_hip_experts_gate_up_silu_mx_f16
    good = [FAKE] * 7 + [5, 4, 16, 96, 64, 6, STREAM]
    refusals(fn, good, {0: [None, FAKE + 8], 1: [None, FAKE + 2], 2: [None, FAKE + 8], 3: [None, FAKE + 2],
                        4: [None, FAKE + 2], 5: [None, FAKE + 2], 6: [None, FAKE + 1], 7: [1 << 31], 8: [65], 9: [1025],
                        10: [95, 1 << 25], 11: [33, 1 << 25], 12: [5], 13: [None]})
    nothing(fn, good, [7, 8, 9, 11])


def workspace(lib, *sizes):
    need = ctypes.c_size_t(99)
    return lib.mote_hip_experts_down_workspace(*sizes, ctypes.byref(need)), need.value


def test_down(lib):
    assert workspace(lib, 0, 4, 16, 64, 96) == (0, 0)
    status, need = workspace(lib, 5, 4, 16, 64, 96)
    assert status == 0 and need > 0
    assert workspace(lib, 5, 4, 16, 65, 96) == (-1, 99)
    assert lib.mote_hip_experts_down_workspace(5, 4, 16, 64, 96, None) == -1
    fn = lib.mote_hip_experts_down_mx_f16
    good = [FAKE] * 9 + [5, 4, 16, 64, 96, 6, FAKE, need, STREAM]
    refusals(fn, good, {0: [None, FAKE + 8], 1: [None, FAKE + 2], 2: [None, FAKE + 8], 3: [None, FAKE + 2],
                        4: [None, FAKE + 2], 5: [None, FAKE + 2], 6: [None, FAKE + 2], 7: [None, FAKE + 2],
                        8: [None, FAKE + 1], 9: [1 << 31], 10: [65], 11: [1025], 12: [33, 1 << 25], 13: [95], 14: [5],
                        15: [None, FAKE + 8], 16: [0, need - 1], 17: [None]})
    nothing(fn, good, [9, 12])


def test_python_calls_refuse_negative_strides():
    from mote_amd import ops

    for fn in (ops.mx_quantize_f16, ops.mx_quantize_f32, ops.mx_dequantize_f16, ops.mx_dequantize_f32):
        with pytest.raises(ValueError):
            fn(FAKE, FAKE, FAKE, 1, 32, 4, STREAM, stride=-32)
    assert ops.mx_value_bytes(96, 4) == 64 and ops.mx_value_bytes(160, 6) == 192 and ops.mx_scale_bytes(160) == 8


@pytest.mark.parametrize("bits", [4, 6])
def test_oracle_codes(bits):
    rng = np.random.default_rng(bits)
    values, scales = mx.random_rows(rng, 3, 160, bits)
    assert values.shape == (3, 256 * bits // 8) and scales.shape == (3, 8)
    codes = mx.unpack(values, bits)
    np.testing.assert_array_equal(mx.pack(codes, bits), values)
    # a row quantised again is what it was, where a block's largest element is the format's
    x = mx.elements(bits)[codes[:, :160]].reshape(3, 5, 32)
    x[:, :, 0] = mx.UP[bits][-1]
    again = mx.read(*mx.quantize(x.reshape(3, 160), bits), bits)[:, :160]
    np.testing.assert_array_equal(again, x.reshape(3, 160))


def test_oracle_4_bits_are_pairs_in_bytes():
    codes = np.arange(128)[None] % 16
    np.testing.assert_array_equal(mx.pack(codes, 4)[0, :8], [0x10, 0x32, 0x54, 0x76, 0x98, 0xBA, 0xDC, 0xFE])
