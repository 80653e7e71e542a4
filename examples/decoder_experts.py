"""The MLP block of a decoder layer with experts, on the library's kernels: fused
add + RMSNorm, the router's projection (Q8_0), the experts' choice and their products on
weights in microscaled 4 bits, and the next layer's add + RMSNorm.

    python examples/decoder_experts.py [--hidden 2048] [--inner 768] [--experts 64] [--top 6] [--tokens 300]

Weights and activations are random.  A prompt's tokens are computed together, then
its last tokens one by one, and the two compared.
"""

from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np

from mote_amd import ops
from mote_amd.device import DeviceBuffer, Stream
from mote_amd.experts import ExpertsMX

EPSILON = 1e-5


def unit_q8_0(rng, n, k):
    """Q8_0 [n, k] whose products of unit inputs are about one."""
    blocks = rng.integers(0, 256, (n * (k // 32), 34), dtype=np.uint8)
    scales = np.abs(rng.standard_normal(len(blocks))) / (74 * np.sqrt(k))
    blocks[:, :2] = scales.astype("<f2").view(np.uint8).reshape(-1, 2)
    return DeviceBuffer.from_array(blocks)


class ExpertsBlock:
    def __init__(self, hidden, inner, experts, top, tokens, stream, bits=6, seed=1):
        rng = np.random.default_rng(seed)
        self.hidden, self.count = hidden, experts
        norm = lambda: DeviceBuffer.from_array((1 + 0.1 * rng.standard_normal(hidden)).astype(np.float16))  # noqa: E731
        self.norm, self.next_norm = norm(), norm()
        self.router = unit_q8_0(rng, experts, hidden)
        self.experts = ExpertsMX(experts, top, hidden, inner, tokens, bits, bias=0.01 * rng.standard_normal(experts))
        draw = lambda n, k: rng.standard_normal((n, k), np.float32) / np.float32(np.sqrt(k))  # noqa: E731
        for e in range(experts):
            self.experts.load(e, draw(inner, hidden), draw(inner, hidden), draw(hidden, inner), stream)
        self.xn, self.y, self.out = (DeviceBuffer(2 * tokens * hidden) for _ in range(3))
        self.logits = DeviceBuffer(4 * tokens * experts)

    def run(self, attended, residual, tokens, stream):
        """The residual grows by attention's and then by the experts' output; `out`
        holds the next layer's input."""
        ops.fused_add_rms_norm_f16(attended, residual, self.norm.ptr, self.xn.ptr, tokens, self.hidden, EPSILON, stream)
        ops.quantized_linear_q8_0_f32(self.xn.ptr, self.router.ptr, self.logits.ptr, tokens, self.count, self.hidden,
                                      stream)
        self.experts.forward(self.xn.ptr, self.logits.ptr, self.y.ptr, tokens, stream)
        ops.fused_add_rms_norm_f16(self.y.ptr, residual, self.next_norm.ptr, self.out.ptr, tokens, self.hidden, EPSILON,
                                   stream)


def run(hidden=2048, inner=768, experts=64, top=6, tokens=300, single=4, bits=6, seed=2):
    """The last `single` tokens' outputs computed with the others and one by one."""
    rng = np.random.default_rng(seed)
    stream = Stream()
    block = ExpertsBlock(hidden, inner, experts, top, tokens, stream, bits)
    attended, residual = (rng.standard_normal((tokens, hidden)).astype(np.float16) for _ in range(2))
    a, r = DeviceBuffer.from_array(attended), DeviceBuffer.from_array(residual)
    block.run(a.ptr, r.ptr, tokens, stream)
    stream.synchronize()
    together = block.out.download(np.float16).reshape(tokens, hidden)[tokens - single:]
    alone = []
    for t in range(tokens - single, tokens):
        a.upload(attended[t])
        r.upload(residual[t])
        block.run(a.ptr, r.ptr, 1, stream)
        stream.synchronize()
        alone.append(block.out.download(np.float16, count=hidden))
    block.experts.free()
    stream.close()
    return together.astype(np.float64), np.array(alone, np.float64)


def main() -> int:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--hidden", type=int, default=2048)
    p.add_argument("--inner", type=int, default=768)
    p.add_argument("--experts", type=int, default=64)
    p.add_argument("--top", type=int, default=6)
    p.add_argument("--tokens", type=int, default=300)
    a = p.parse_args()
    together, alone = run(a.hidden, a.inner, a.experts, a.top, a.tokens)
    off = np.sqrt(((together - alone) ** 2).mean() / (together ** 2).mean())
    print(f"tokens one by one differ from the same in a prompt by {off:.5f} of the output's size")
    return 0


if __name__ == "__main__":
    sys.exit(main())
