"""The attention block of a decoder layer, from prompts to generated tokens, on
the library's kernels: RMSNorm, the q / k / v projections (Q4_0), RoPE, the keys
and values into the 8-bit cache, attention of the prompts over their own keys and
of the generated tokens over the cache, and the output projection.

    python examples/decoder_attention.py [--hidden 4096] [--heads 32] [--kv-heads 8] [--steps 16]

Weights and activations are random.  At the end the last tokens of every sequence
are computed again as a prompt, from unrounded keys and values, and compared.
"""

from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np

from mote_amd import ops
from mote_amd.device import DeviceBuffer, Stream
from mote_amd.kv_cache import KVCacheQ8

EPSILON = 1e-5
THETA = 500000.0


def unit_q4_0(rng, n, k):
    """Q4_0 [n, k] whose products of unit inputs are about one."""
    blocks = rng.integers(0, 256, (n * (k // 32), 18), dtype=np.uint8)
    scales = np.abs(rng.standard_normal(len(blocks))) / (4.6 * np.sqrt(k))
    blocks[:, :2] = scales.astype("<f2").view(np.uint8).reshape(-1, 2)
    return DeviceBuffer.from_array(blocks)


class AttentionBlock:
    def __init__(self, hidden, heads, kv_heads, head_dim, sequences, context, rows, seed=1):
        rng = np.random.default_rng(seed)
        self.hidden, self.heads, self.kv_heads, self.head_dim = hidden, heads, kv_heads, head_dim
        self.width, self.kv_width = heads * head_dim, kv_heads * head_dim
        self.norm = DeviceBuffer.from_array((1 + 0.1 * rng.standard_normal(hidden)).astype(np.float16))
        self.wq = unit_q4_0(rng, self.width, hidden)
        self.wk, self.wv = (unit_q4_0(rng, self.kv_width, hidden) for _ in range(2))
        self.wo = unit_q4_0(rng, hidden, self.width)
        blocks = sequences * -(-context // ops.KV_BLOCK_TOKENS)
        self.cache = KVCacheQ8(blocks, kv_heads, head_dim, sequences, context)
        half = lambda n: DeviceBuffer(2 * rows * n)  # noqa: E731
        self.xn, self.q, self.k, self.v = half(hidden), half(self.width), half(self.kv_width), half(self.kv_width)
        self.attended, self.y = half(self.width), half(hidden)
        self.positions = DeviceBuffer(8 * rows)
        self.cos, self.sin = (DeviceBuffer(4 * rows * (head_dim // 2)) for _ in range(2))
        self.offsets = DeviceBuffer(4 * (sequences + 1))
        self.workspace = DeviceBuffer(0)

    def project(self, x, counts, first, stream):
        """q, k and v of packed rows x whose sequences go on at first[i]."""
        rows, h = sum(counts), self.hidden
        at = np.concatenate([f + np.arange(n) for f, n in zip(first, counts)]).astype(np.int64)
        self.positions.upload(at)
        ops.rope_tables_f32(self.positions.ptr, self.cos.ptr, self.sin.ptr, rows, self.head_dim, THETA, stream)
        ops.rms_norm_f16(x, self.norm.ptr, self.xn.ptr, rows, h, EPSILON, stream)
        ops.quantized_linear_q4_0_f16(self.xn.ptr, self.wq.ptr, self.q.ptr, rows, self.width, h, stream)
        ops.quantized_linear_q4_0_f16(self.xn.ptr, self.wk.ptr, self.k.ptr, rows, self.kv_width, h, stream)
        ops.quantized_linear_q4_0_f16(self.xn.ptr, self.wv.ptr, self.v.ptr, rows, self.kv_width, h, stream)
        ops.rope_qk_f16(self.q.ptr, self.k.ptr, self.cos.ptr, self.sin.ptr, self.q.ptr, self.k.ptr, rows, self.heads,
                        self.kv_heads, self.head_dim, self.head_dim, ops.HALF_SPLIT, stream)

    def output(self, rows, stream):
        ops.quantized_linear_q4_0_f16(self.attended.ptr, self.wo.ptr, self.y.ptr, rows, self.hidden, self.width, stream)

    def prompts(self, sequences, x, counts, stream):
        """New sequences' prompts: into the cache, and attention over their own keys."""
        self.project(x, counts, [0] * len(counts), stream)
        if sequences is not None:
            self.cache.append(sequences, self.k.ptr, self.v.ptr, counts, stream)
        self.offsets.upload(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        rows = sum(counts)
        shape = (len(counts), rows, rows, max(counts), self.heads, self.kv_heads, self.head_dim)
        need = ops.prompt_attention_workspace(*shape)
        if need > self.workspace.nbytes:
            stream.synchronize()
            self.workspace = DeviceBuffer(need)
        ops.prompt_attention_f16(self.q.ptr, self.k.ptr, self.v.ptr, self.attended.ptr, self.offsets.ptr, None, *shape,
                                 self.head_dim ** -0.5, self.workspace.ptr, self.workspace.nbytes, stream)
        self.output(rows, stream)

    def tokens(self, sequences, x, counts, stream):
        """The next tokens of known sequences, over the cache."""
        self.project(x, counts, [self.cache.length(s) for s in sequences], stream)
        self.cache.append(sequences, self.k.ptr, self.v.ptr, counts, stream)
        self.cache.attend(sequences, self.q.ptr, self.attended.ptr, self.heads, counts, stream)
        self.output(sum(counts), stream)


def run(hidden=4096, heads=32, kv_heads=8, head_dim=128, prompts=(300, 45, 1000, 7), steps=16, seed=2):
    """The largest difference of the last step's output from the same computed
    as a prompt, over the output's root mean square."""
    rng = np.random.default_rng(seed)
    total = [n + steps for n in prompts]
    x = [rng.standard_normal((n, hidden)).astype(np.float16) for n in total]
    stream = Stream()
    block = AttentionBlock(hidden, heads, kv_heads, head_dim, len(prompts), max(total), sum(total))
    upload = lambda rows: DeviceBuffer.from_array(np.concatenate(rows))  # noqa: E731
    sequences = [block.cache.open() for _ in prompts]
    first = upload([r[:n] for r, n in zip(x, prompts)])
    block.prompts(sequences, first.ptr, list(prompts), stream)
    for step in range(steps):
        now = upload([r[n + step:n + step + 1] for r, n in zip(x, prompts)])
        block.tokens(sequences, now.ptr, [1] * len(prompts), stream)
        stream.synchronize()
    got = block.y.download(np.float16, count=len(prompts) * hidden).reshape(len(prompts), hidden)
    whole = upload(x)
    block.prompts(None, whole.ptr, total, stream)
    stream.synchronize()
    rows = np.cumsum(total) - 1
    want = block.y.download(np.float16, count=sum(total) * hidden).reshape(-1, hidden)[rows]
    got, want = got.astype(np.float64), want.astype(np.float64)
    stream.close()
    return float(np.abs(got - want).max() / np.sqrt((want ** 2).mean()))


def main() -> int:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--hidden", type=int, default=4096)
    p.add_argument("--heads", type=int, default=32)
    p.add_argument("--kv-heads", type=int, default=8)
    p.add_argument("--head-dim", type=int, default=128)
    p.add_argument("--steps", type=int, default=16)
    a = p.parse_args()
    off = run(a.hidden, a.heads, a.kv_heads, a.head_dim, steps=a.steps)
    print(f"generated tokens over the 8-bit cache differ from the same as a prompt by {off:.4f} of the output's size")
    return 0


if __name__ == "__main__":
    sys.exit(main())
