"""The MLP of a mixture-of-experts layer on weights in microscaled 4 bits: the
calls from router logits to the layer's output
(``mote_hip_route_experts_*``, ``mote_hip_plan_experts``, ``mote_hip_mx_quantize_f16``,
``mote_hip_experts_gate_up_silu_mx_f16`` and ``mote_hip_experts_down_mx_f16`` of
include/mote_hip.h) and the memory they need.
"""

from __future__ import annotations

import numpy as np

from . import ops
from ._ffi import check, lib
from .device import DeviceBuffer


class ExpertsMX:
    """``experts`` MLPs, silu(x gate^T) (x up^T) down^T, of which each token takes
    the ``top`` best by its logits.

    ``bits``: of the activations, 4 or 6.  ``score``, ``groups``, ``top_groups``,
    ``group_best``, ``renormalize`` and ``scale`` as for ``ops.route_experts_f32``.
    Weights come by ``load``, or, already in 4 bits, to ``gate_up`` and ``down`` and their scales
    (an expert's gate rows, its up rows, the next expert's; down rows likewise); what an expert
    computes before is undefined.  All memory is taken here, for up to ``max_tokens`` tokens:
    ``forward`` allocates nothing, does not wait, and can be captured.  Its calls share that memory, so they follow
    each other on one stream (or are ordered by the caller).
    """

    def __init__(self, experts: int, top: int, hidden: int, inner: int, max_tokens: int, bits: int = 6,
                 score: int = ops.SOFTMAX, bias=None, groups: int = 1, top_groups: int = 1, group_best: int = 2,
                 renormalize: bool = True, scale: float = 1.0) -> None:
        if experts < 1 or not 1 <= top <= experts or max_tokens < 1:
            raise ValueError("an expert, a choice of no more than there are, and a token at least")
        if experts > 1024 or top > 64 or max_tokens > (1 << 26) - 4 or max_tokens * top > 1 << 30:
            raise ValueError("up to 1024 experts, 64 of a token, 2^26 - 4 tokens and 2^30 choices")
        if any(n < 32 or n % 32 or n > 1 << 24 for n in (hidden, inner)):
            raise ValueError("hidden and inner elements are multiples of 32, up to 2^24")
        if score not in (ops.SOFTMAX, ops.SIGMOID) or group_best not in (1, 2) or not abs(scale) <= 3.4028234663852886e38:
            raise ValueError("scores of softmax or sigmoid, groups by one or two choices, a finite scale")
        if groups < 1 or experts % groups or not 1 <= top_groups <= groups:
            raise ValueError("groups of as many experts each, and one of them at least")
        if top > top_groups * (experts // groups):
            raise ValueError("no more choices than the groups leave experts")
        if bits not in (4, 6):
            raise ValueError("activations of 4 or 6 bits")
        if bias is not None and np.shape(bias) != (experts,):
            raise ValueError("a bias for each expert")
        self.experts, self.top, self.hidden, self.inner = experts, top, hidden, inner
        self.max_tokens, self.bits = max_tokens, bits
        self._routing = dict(score=score, groups=groups, top_groups=top_groups, group_best=group_best,
                             renormalize=renormalize, scale=scale)
        self._bias = None if bias is None else DeviceBuffer.from_array(np.asarray(bias, np.float32))
        self.gate_up, self.gate_up_scales = self._rows(experts * 2 * inner, hidden, 4)
        self.down, self.down_scales = self._rows(experts * hidden, inner, 4)
        pairs = max_tokens * top
        self.ids, self.weights, self._plan = (DeviceBuffer(4 * pairs) for _ in range(3))
        self._offsets = DeviceBuffer(4 * (experts + 1))
        self._x, self._x_scales = self._rows(max_tokens, hidden, bits)
        self._h = DeviceBuffer(2 * pairs * inner)
        self._h_values, self._h_scales = self._rows(pairs, inner, bits)
        self._workspace = DeviceBuffer(ops.experts_down_workspace(max_tokens, top, experts, hidden, inner))

    @staticmethod
    def _rows(rows, features, bits):
        return (DeviceBuffer(rows * ops.mx_value_bytes(features, bits)),
                DeviceBuffer(rows * ops.mx_scale_bytes(features)))

    def load(self, expert: int, gate, up, down, stream) -> None:
        """An expert's weights from arrays gate and up [inner, hidden] and down
        [hidden, inner], rounded to 4 bits.  Waits for the stream."""
        if not 0 <= expert < self.experts:
            raise ValueError(f"no expert {expert}")
        shapes = [(self.inner, self.hidden)] * 2 + [(self.hidden, self.inner)]
        arrays = [np.ascontiguousarray(a, np.float32) for a in (gate, up, down)]
        for a, shape in zip(arrays, shapes):
            if a.shape != shape:
                raise ValueError(f"weights of shape {a.shape}, not {shape}")
        held = []  # until the stream has been waited for
        for a, (values, scales), first in (
                (arrays[0], (self.gate_up, self.gate_up_scales), 2 * expert * self.inner),
                (arrays[1], (self.gate_up, self.gate_up_scales), (2 * expert + 1) * self.inner),
                (arrays[2], (self.down, self.down_scales), expert * self.hidden)):
            rows, features = a.shape
            held.append(DeviceBuffer.from_array(a))
            ops.mx_quantize_f32(held[-1].ptr, values.ptr + first * ops.mx_value_bytes(features, 4),
                                scales.ptr + first * ops.mx_scale_bytes(features), rows, features, 4, stream)
        check(lib().mote_hip_stream_synchronize(ops._s(stream)), "synchronize stream")

    def forward(self, x: int, logits: int, y: int, tokens: int, stream, logits_f16: bool = False, stride=None) -> None:
        """y [tokens, hidden] (f16) of x (f16, rows `stride` elements apart) and router logits
        [tokens, experts] (f32, or f16), all device addresses."""
        if not 0 <= tokens <= self.max_tokens:
            raise ValueError(f"up to {self.max_tokens} tokens")
        sizes = (tokens, self.top, self.experts, self.hidden, self.inner)
        route = ops.route_experts_f16 if logits_f16 else ops.route_experts_f32
        route(logits, self._bias.ptr if self._bias else None, self.ids.ptr, self.weights.ptr, tokens, self.experts,
              self.top, stream, **self._routing)
        ops.plan_experts(self.ids.ptr, self._offsets.ptr, self._plan.ptr, tokens, self.top, self.experts, stream)
        ops.mx_quantize_f16(x, self._x.ptr, self._x_scales.ptr, tokens, self.hidden, self.bits, stream, stride)
        ops.experts_gate_up_silu_mx_f16(self._x.ptr, self._x_scales.ptr, self.gate_up.ptr, self.gate_up_scales.ptr,
                                        self._offsets.ptr, self._plan.ptr, self._h.ptr, *sizes, self.bits, stream)
        ops.mx_quantize_f16(self._h.ptr, self._h_values.ptr, self._h_scales.ptr, tokens * self.top, self.inner,
                            self.bits, stream)
        ops.experts_down_mx_f16(self._h_values.ptr, self._h_scales.ptr, self.down.ptr, self.down_scales.ptr,
                                self.ids.ptr, self._offsets.ptr, self._plan.ptr, self.weights.ptr, y, *sizes, self.bits,
                                self._workspace.ptr, self._workspace.nbytes, stream)

    def free(self) -> None:
        """Gives the memory back; no call may be under way."""
        for b in (self.gate_up, self.gate_up_scales, self.down, self.down_scales, self.ids, self.weights, self._plan,
                  self._offsets, self._x, self._x_scales, self._h, self._h_values, self._h_scales, self._workspace):
            b.free()
        if self._bias:
            self._bias.free()
