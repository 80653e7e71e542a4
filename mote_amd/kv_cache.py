"""An 8-bit key/value cache for many sequences: blocks of 32 tokens given out
from one pool, and the calls that write and read them
(``mote_hip_kv_cache_append_q8``, ``mote_hip_kv_cache_read_q8_f16`` and
``mote_hip_cache_attention_q8_f16`` of include/mote_hip.h).

:class:`BlockTable` is the host's book-keeping alone; :class:`KVCacheQ8` adds the
device memory.  The small arrays that describe a call (offsets, lengths, the
block table) are uploaded by each call, which first waits for the stream of the
call before (so calls may use different streams; one given by its handle must
live until the next call).  That costs the host some 70 us a call: a program that
captures graphs, cannot wait, or has the same sequences in many layers keeps its
own on the device and calls ``mote_amd.ops`` directly.
"""

from __future__ import annotations

import operator

import numpy as np

from . import ops
from ._ffi import check, lib
from .device import DeviceBuffer


class CacheFull(RuntimeError):
    """The pool has no block left, or a sequence no room in its table."""


def _integers(values) -> list[int]:
    """A call's numbers, in whatever form they come (numpy takes a tuple of two
    indices for a row and a column)."""
    return [operator.index(v) for v in values]


class BlockTable:
    """Which blocks hold the tokens of each sequence."""

    def __init__(self, blocks: int, max_sequences: int, max_context: int) -> None:
        if blocks < 1 or max_sequences < 1 or max_context < 1:
            raise ValueError("a cache needs a block, a sequence and a token at least")
        self.blocks = blocks
        self.width = -(-max_context // ops.KV_BLOCK_TOKENS)
        self.table = np.full((max_sequences, self.width), -1, np.int32)
        self.lengths = np.zeros(max_sequences, np.int64)
        self._open = np.zeros(max_sequences, bool)
        self._free = list(range(blocks - 1, -1, -1))

    @property
    def free_blocks(self) -> int:
        return len(self._free)

    def open(self) -> int:
        """A new sequence's number."""
        idle = np.flatnonzero(~self._open)
        if idle.size == 0:
            raise CacheFull("every sequence is in use")
        self._open[idle[0]] = True
        return int(idle[0])

    def close(self, sequence: int) -> None:
        """Ends a sequence; its blocks return to the pool."""
        self._known([sequence])
        row = self.table[sequence]
        self._free.extend(int(b) for b in row[row >= 0][::-1])
        row[:] = -1
        self.lengths[sequence] = 0
        self._open[sequence] = False

    def reserve(self, sequences, counts) -> None:
        """Blocks for counts[i] more tokens of sequences[i]; all or none."""
        self._known(sequences)
        need = []
        for s, n in zip(sequences, counts):
            if n < 0:
                raise ValueError("a negative number of tokens")
            held = int((self.table[s] >= 0).sum())
            last = -(-int(self.lengths[s] + n) // ops.KV_BLOCK_TOKENS)
            if last > self.width:
                raise CacheFull(f"sequence {s} would pass {self.width * ops.KV_BLOCK_TOKENS} tokens")
            need.append((s, held, max(last, held)))
        if sum(last - held for _, held, last in need) > len(self._free):
            raise CacheFull(f"{len(self._free)} blocks are free")
        for s, held, last in need:
            for b in range(held, last):
                self.table[s, b] = self._free.pop()

    def advance(self, sequences, counts) -> None:
        for s, n in zip(sequences, counts):
            self.lengths[s] += n

    def truncate(self, sequence: int, length: int) -> None:
        """Forgets the tokens from `length` on (drafts that were not taken).  What
        they made of the block that `length` lies in stays: its scales, which are
        NaN where one of them was not finite."""
        self._known([sequence])
        if not 0 <= length <= self.lengths[sequence]:
            raise ValueError(f"sequence {sequence} holds {self.lengths[sequence]} tokens")
        keep = -(-length // ops.KV_BLOCK_TOKENS)
        row = self.table[sequence]
        self._free.extend(int(b) for b in row[keep:][row[keep:] >= 0][::-1])
        row[keep:] = -1
        self.lengths[sequence] = length

    def _known(self, sequences) -> None:
        if len(set(sequences)) != len(sequences):
            raise ValueError("a sequence is named twice")
        for s in sequences:
            if not 0 <= s < len(self._open) or not self._open[s]:
                raise ValueError(f"no open sequence {s}")


class KVCacheQ8:
    """The cache of one attention layer.

    ``k``, ``v``, ``q`` and ``out`` are device addresses of packed f16 rows: the
    rows of ``sequences[0]`` first, ``counts[0]`` of them, and so on.
    ``sequences``, ``counts`` and ``first`` are integers in any iterable.
    """

    def __init__(self, blocks: int, kv_heads: int, head_dim: int, max_sequences: int, max_context: int) -> None:
        if kv_heads < 1 or head_dim < 8 or head_dim % 8 != 0 or head_dim > 256:
            raise ValueError("heads of 8 to 256 dimensions, a multiple of 8")
        self.kv_heads, self.head_dim = kv_heads, head_dim
        self.blocks = BlockTable(blocks, max_sequences, max_context)
        self.cache = DeviceBuffer(blocks * 2 * kv_heads * ops.kv_plane_bytes(head_dim))
        self.scales = DeviceBuffer(blocks * 2 * kv_heads * 4)
        self._table = DeviceBuffer(self.blocks.table.nbytes)
        self._offsets = DeviceBuffer(4 * (max_sequences + 1))
        self._second = DeviceBuffer(4 * max_sequences)
        self._workspace = DeviceBuffer(0)
        self._last = None  # the stream that may still use them

    def open(self) -> int:
        return self.blocks.open()

    def close(self, sequence: int) -> None:
        self.blocks.close(sequence)

    def truncate(self, sequence: int, length: int) -> None:
        self.blocks.truncate(sequence, length)

    def length(self, sequence: int) -> int:
        return int(self.blocks.lengths[sequence])

    def append(self, sequences, k: int, v: int, counts, stream, strides=None) -> None:
        """The next counts[i] tokens of sequences[i]."""
        sequences, counts = _integers(sequences), _integers(counts)
        if len(sequences) != len(counts):
            raise ValueError("one count for each sequence")
        self.blocks.reserve(sequences, counts)
        self._upload(sequences, counts, self.blocks.lengths[sequences], stream)
        ops.kv_cache_append_q8(k, v, self._offsets.ptr, self._second.ptr, self._table.ptr, self.cache.ptr,
                               self.scales.ptr, len(sequences), sum(counts), *self._shape(), stream, strides)
        self.blocks.advance(sequences, counts)

    def read(self, sequences, k: int, v: int, counts, first, stream, strides=None) -> None:
        """counts[i] tokens of sequences[i] from first[i] on, in f16."""
        sequences, counts, first = _integers(sequences), _integers(counts), _integers(first)
        if not len(sequences) == len(counts) == len(first):
            raise ValueError("one count and one first token for each sequence")
        self.blocks._known(sequences)
        for s, n, at in zip(sequences, counts, first):
            if n < 0 or at < 0 or at + n > self.blocks.lengths[s]:
                raise ValueError(f"sequence {s} holds {self.blocks.lengths[s]} tokens")
        self._upload(sequences, counts, first, stream)
        ops.kv_cache_read_q8_f16(self.cache.ptr, self.scales.ptr, self._offsets.ptr, self._second.ptr,
                                 self._table.ptr, k, v, len(sequences), sum(counts), *self._shape(), stream,
                                 strides)

    def attend(self, sequences, q: int, out: int, q_heads: int, counts, stream, scale=None, window: int = 0,
               strides=None) -> None:
        """Attention of the last counts[i] tokens of sequences[i], their own keys
        already appended.  `scale` None: 1 / sqrt(head_dim)."""
        sequences, counts = _integers(sequences), _integers(counts)
        if len(sequences) != len(counts):
            raise ValueError("one count for each sequence")
        self.blocks._known(sequences)
        lengths = self.blocks.lengths[sequences]
        for s, n in zip(sequences, counts):
            if not 0 <= n <= self.blocks.lengths[s]:
                raise ValueError(f"sequence {s} holds {self.blocks.lengths[s]} tokens")
        if not len(sequences) or not sum(counts):
            return
        self._upload(sequences, counts, lengths, stream)
        shape = (len(sequences), sum(counts), max(counts), int(lengths.max()), q_heads, self.kv_heads,
                 self.head_dim)
        need = ops.cache_attention_workspace(*shape)
        if need > self._workspace.nbytes:  # nothing uses the old one: the upload has waited
            self._workspace = DeviceBuffer(need)
        ops.cache_attention_q8_f16(
            q, self.cache.ptr, self.scales.ptr, self._offsets.ptr, self._second.ptr, self._table.ptr, out, *shape,
            self.blocks.width, self.blocks.blocks, self.head_dim ** -0.5 if scale is None else scale,
            self._workspace.ptr, self._workspace.nbytes, stream, window=window, strides=strides)

    def free(self) -> None:
        self._wait()
        for b in (self.cache, self.scales, self._table, self._offsets, self._second, self._workspace):
            b.free()

    def _shape(self):
        return self.kv_heads, self.head_dim, self.blocks.width, self.blocks.blocks

    def _wait(self) -> None:
        handle = getattr(self._last, "handle", self._last)
        if handle:  # a closed stream has been waited for
            check(lib().mote_hip_stream_synchronize(handle), "synchronize stream")
        self._last = None

    def _upload(self, sequences, counts, second, stream) -> None:
        self._wait()
        self._last = stream
        self._offsets.upload(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        self._second.upload(np.asarray(second, np.int32))
        self._table.upload(self.blocks.table[sequences])
