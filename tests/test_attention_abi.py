"""What the attention and cache entry points refuse, and the calls that have
nothing to do (CPU: every check comes before any device work, so stand-in
pointers are never followed)."""

from __future__ import annotations

import ctypes
import os

import pytest

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


# sequences, query tokens, key tokens, most keys, heads, key heads, head size
PROMPT = [2, 60, 70, 40, 8, 2, 64]
PROMPT_CALL = [FAKE] * 6 + PROMPT + [512, 128, 128, 512] + [0.125, 1, 0, FAKE, 1 << 40, STREAM]


def test_prompt_attention_refusals(lib):
    fn = lib.mote_hip_prompt_attention_f16
    bad = {0: [None, FAKE + 1], 1: [None, FAKE + 1], 2: [None, FAKE + 1], 3: [None, FAKE + 1], 4: [None, FAKE + 2],
           5: [None, FAKE + 2],  # no key offsets, but other key rows than query rows
           6: [1 << 31], 7: [1 << 31], 8: [1 << 31], 9: [1 << 31], 10: [7, 1 << 16], 11: [0, 3, 16],
           12: [12, 264], 16: [511], 17: [0.0, -1.0, NAN, INF, 3e38], 18: [2, -1], 22: [None]}
    refusals(fn, PROMPT_CALL, bad)
    args = list(PROMPT_CALL)
    args[18], args[19] = 0, 5  # a window without causal
    assert fn(*args) == -1


def test_prompt_attention_of_nothing(lib):
    for at in (6, 7, 10, 12):
        args = list(PROMPT_CALL)
        args[at] = 0
        if at == 10:
            args[11] = 0
        assert lib.mote_hip_prompt_attention_f16(*args) == 0, at


def workspace(fn, *sizes):
    need = ctypes.c_size_t(99)
    return fn(*sizes, ctypes.byref(need)), need.value


def test_prompt_attention_workspace(lib):
    fn = lib.mote_hip_prompt_attention_workspace
    assert workspace(fn, 1, 100000, 100000, 100000, 32, 8, 128) == (0, 0)  # rows enough
    status, few = workspace(fn, 1, 1, 8000, 8000, 8, 8, 128)
    assert status == 0 and few > 0
    assert workspace(fn, 0, 0, 0, 0, 32, 8, 128) == (0, 0)
    assert workspace(fn, 1, 1, 1, 1, 5, 2, 128) == (-1, 0)
    assert workspace(fn, 1, 1, 1, 1, 4, 2, 100) == (-1, 0)
    assert fn(1, 1, 1, 1, 4, 2, 64, None) == -1
    call = [FAKE] * 6 + [1, 1, 8000, 8000, 8, 8, 128, 1024, 1024, 1024, 1024, 0.1, 1, 0]
    for work, size in ((None, few), (FAKE, few - 1), (FAKE + 8, few), (FAKE, 0)):
        assert lib.mote_hip_prompt_attention_f16(*call, work, size, STREAM) == -1


CACHE_CALL = [FAKE] * 7 + [3, 40, 2, 64, 128, 128, 10, 100, STREAM]


@pytest.mark.parametrize("name", ["append", "read"])
def test_cache_refusals(lib, name):
    if name == "append":  # k, v, offsets, positions, table, cache, scales
        fn, half, word, cache = lib.mote_hip_kv_cache_append_q8, (0, 1), (2, 3, 4, 6), 5
    else:  # cache, scales, offsets, positions, table, k, v
        fn, half, word, cache = lib.mote_hip_kv_cache_read_q8_f16, (5, 6), (1, 2, 3, 4), 0
    bad = {i: [None] for i in range(7)} | {15: [None], 10: [12, 264], 8: [1 << 31], 7: [1 << 31], 9: [1 << 16],
                                           13: [1 << 26], 14: [1 << 31]}
    for i in half:
        bad[i] = [None, FAKE + 1]
    for i in word:
        bad[i] = [None, FAKE + 2]
    bad[cache] = [None, FAKE + 8]
    if name == "read":
        bad[11], bad[12] = [127], [127]
    refusals(fn, CACHE_CALL, bad)
    for at in (7, 8, 9, 10):
        args = list(CACHE_CALL)
        args[at] = 0
        assert fn(*args) == 0, at


# q, cache, scales, query offsets, lengths, table, output; sequences, query tokens,
# most queries, most context, heads, key heads, head size; strides, table, cache
ATTEND_CALL = [FAKE] * 7 + [2, 6, 4, 300, 8, 2, 64, 512, 512, 10, 100, 0.125, 0, FAKE, 1 << 40, STREAM]


def test_cache_attention_refusals(lib):
    fn = lib.mote_hip_cache_attention_q8_f16
    bad = {0: [None, FAKE + 1], 1: [None, FAKE + 8], 2: [None, FAKE + 2], 3: [None, FAKE + 2],
           4: [None, FAKE + 2], 5: [None, FAKE + 2], 6: [None, FAKE + 1], 7: [1 << 31], 8: [1 << 31], 9: [1 << 31],
           10: [1 << 31], 11: [7, 1 << 16], 12: [0, 3, 16], 13: [12, 264], 15: [511], 16: [1 << 26], 17: [1 << 31],
           18: [0.0, -1.0, NAN, INF, 3e38], 22: [None]}
    refusals(fn, ATTEND_CALL, bad)
    for tokens, most in ((3, 1), (2, 2)):  # no offsets: one query a sequence
        args = list(ATTEND_CALL)
        args[3], args[8], args[9] = None, tokens, most
        assert fn(*args) == -1
    for at in (7, 8, 9, 11, 13):
        args = list(ATTEND_CALL)
        args[at] = 0
        if at == 11:
            args[12] = 0
        assert fn(*args) == 0, at


def test_cache_attention_workspace(lib):
    fn = lib.mote_hip_cache_attention_workspace
    assert workspace(fn, 4096, 4096, 1, 64, 8, 8, 128) == (0, 0)
    status, long = workspace(fn, 1, 1, 1, 100000, 8, 2, 128)
    assert status == 0 and long > 0
    assert workspace(fn, 1, 1, 1, 1, 5, 2, 128) == (-1, 0)
    assert fn(1, 1, 1, 1, 4, 2, 64, None) == -1
    call = [FAKE] * 7 + [1, 1, 1, 100000, 8, 2, 128, 1024, 1024, 4000, 5000, 0.1, 0]
    for work, size in ((None, long), (FAKE, long - 1), (FAKE + 8, long), (FAKE, 0)):
        assert lib.mote_hip_cache_attention_q8_f16(*call, work, size, STREAM) == -1


def test_wrappers_raise(lib):
    from mote_amd import HipError, ops

    with pytest.raises(HipError, match="prompt attention"):
        ops.prompt_attention_f16(FAKE, FAKE, FAKE, FAKE, FAKE, None, 1, 4, 4, 4, 3, 2, 64, 0.1, 0, 0, STREAM)
    with pytest.raises(HipError, match="cache attention"):
        ops.cache_attention_workspace(1, 1, 1, 10, 4, 2, 36)
    assert ops.kv_plane_bytes(128) == 4096 and ops.kv_plane_bytes(40) == 2048
