"""Sizes past what the attention's launches can number are refused (CPU: every
check comes before any device work)."""

from __future__ import annotations

import os

import pytest

FAKE, STREAM = 0x10000, 0x20000


@pytest.fixture(scope="module")
def lib():
    from mote_amd import _ffi

    if not os.path.exists(_ffi.LIBRARY):
        from mote_amd import build

        build.build()
    return _ffi.lib()


def test_cache_attention_workgroups(lib):
    """2^30 sequences of four key heads; of two with three tiles of 32 rows; 2^26 of 64
    tiles of 128."""
    tail = [1024, 1024, 1, 100, 0.125, 0, None, 0, STREAM]
    for sizes in ([1 << 30, 1, 1, 32, 4, 4, 64], [1 << 30, 1, 90, 32, 2, 2, 64], [1 << 26, 1, 1 << 12, 32, 2, 1, 64]):
        assert lib.mote_hip_cache_attention_q8_f16(*[FAKE] * 7, *sizes, *tail) == -1, sizes


@pytest.mark.parametrize("window", [-1, -(1 << 40)])
def test_negative_windows(lib, window):
    """As a number without sign they would be larger than any context: no window."""
    from mote_amd import ops

    with pytest.raises(ValueError, match="window"):
        ops.prompt_attention_f16(FAKE, FAKE, FAKE, FAKE, FAKE, None, 1, 4, 4, 4, 4, 2, 64, 0.1, 0, 0, STREAM,
                                 window=window)
    with pytest.raises(ValueError, match="window"):
        ops.cache_attention_q8_f16(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1, 4, 4, 100, 4, 2, 64, 10, 100, 0.1, 0, 0,
                                   STREAM, window=window)
