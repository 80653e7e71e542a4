"""Attention and the 8-bit cache in numpy, from their definitions: attention in
64 bits with a bound on what f32 sums and f16 weights may differ by, the cache's
bytes in the f32 steps that define them."""

from __future__ import annotations

import numpy as np

BLOCK = 32


def attend(q, k, v, scale, causal=True, window=0):
    """One sequence: q [n, heads, d], k and v [t, kv_heads, d] (any float type).
    Returns (o, bound) in float64, both [n, heads, d].

    The bound: the output's rounding to f16 (2^-11 of it, 2^-25 where it is
    subnormal); each weight's rounding to f16 (2^-11); its exponent's error,
    from d products added in f32 (d 2^-24 of their absolute sum) and three
    roundings of the scaled score, once in the weight and once in their sum; the
    sum over t keys in f32 (t 2^-23); weights below 2^-22 of the row's largest
    round with an error of 2^-33 of it; all but the first times sum_j w_j |v_j|."""
    n, heads, d = q.shape
    t, kv_heads = k.shape[:2]
    group = heads // kv_heads
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    o = np.zeros((n, heads, d))
    bound = np.zeros((n, heads, d))
    at = np.arange(n)[:, None] + (t - n)
    j = np.arange(t)[None, :]
    sees = np.ones((n, t), bool)
    if causal:
        sees = j <= at
        if window:
            sees &= j > at - window
    some = sees.any(1)
    if not some.any():
        return o, bound
    mask = sees[some]
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = np.where(mask, (q[some, h] @ kh.T) * scale, -np.inf)
        size = np.where(mask, (np.abs(q[some, h]) @ np.abs(kh).T) * scale, 0.0).max(1)
        most = np.abs(np.where(mask, s, 0.0)).max(1)
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        o[some, h] = w @ vh
        large = np.stack([np.abs(vh[m]).max() for m in mask]) if window else np.maximum.accumulate(
            np.abs(vh).max(1))[mask.shape[1] - 1 - mask[:, ::-1].argmax(1)]
        reach = w @ np.abs(vh) + (2.0**-33 * mask.sum(1) * large)[:, None]
        off = ((d * size + 3 * most + 3) * 2.0**-23)[:, None]
        bound[some, h] = 2.0**-11 * np.abs(o[some, h]) + reach * (2.0**-11 + 2 * off + t * 2.0**-23) + 2.0**-24
    return o, bound


def assert_within(got, want, bound, what=""):
    got = np.asarray(got, dtype=np.float64)
    assert got.shape == want.shape
    err = np.abs(got - want)
    bad = ~(err <= bound)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} out of bound, first {i}: got {got[i]}, "
                             f"want {want[i]} +- {bound[i]}")


# --- the cache ------------------------------------------------------------------


def padded(d: int) -> int:
    return -(-d // 32) * 32


def byte_of(which: int, t, d):
    """Byte of element (token t of the block, dimension d) of a key (0) or value
    (1) plane."""
    c = d // 32
    if which == 0:
        return (((c * 4 + d % 32 // 8) * 16 + t % 16) * 2 + t // 16) * 8 + d % 8
    return (((c * 4 + t % 16 // 4) * 16 + d % 16) * 2 + d % 32 // 16) * 8 + 4 * (t // 16) + t % 4


def plane_index(which: int, d: int) -> np.ndarray:
    """[32, d] byte numbers of a plane."""
    t, x = np.meshgrid(np.arange(BLOCK), np.arange(d), indexing="ij")
    return byte_of(which, t, x)


class Cache:
    """The cache on the host: bytes [blocks, heads, 2, 32 P], scales f32."""

    def __init__(self, blocks, heads, d, rng=None):
        self.heads, self.d = heads, d
        shape = (blocks, heads, 2, BLOCK * padded(d))
        if rng is None:
            self.bytes = np.full(shape, 128, np.uint8)
            self.scales = np.zeros(shape[:3], np.float32)
        else:
            self.bytes = rng.integers(1, 256, shape, dtype=np.uint8)
            self.scales = rng.uniform(0.005, 0.02, shape[:3]).astype(np.float32)
        self.index = [plane_index(w, d) for w in (0, 1)]

    def append(self, x, which, table, position):
        """x [n, heads, d] f16 as tokens position .. of the sequence whose blocks
        are `table`."""
        x = np.asarray(x, np.float16).astype(np.float32)
        if len(x) == 0:
            return
        one = np.float32(1.0)
        for block in range(position // BLOCK, -(-(position + len(x)) // BLOCK)):
            if block >= len(table) or not 0 <= table[block] < len(self.bytes):
                continue
            first, last = max(position, block * BLOCK), min(position + len(x), (block + 1) * BLOCK)
            new = x[first - position:last - position]
            for h in range(self.heads):
                at = (table[block], h, which)
                old = self.scales[at] if first % BLOCK else np.float32(0.0)
                finite = np.isfinite(new[:, h]).all() and np.isfinite(old)
                need = np.abs(new[:, h]).max() / np.float32(127.0) if finite else np.float32("nan")
                scale = np.maximum(old, need) if finite else np.float32("nan")
                inverse = one / scale if scale > 0 else np.float32(0.0)
                plane = self.bytes[at]
                if first % BLOCK == 0:
                    plane[:] = 128  # zeros in the slots not written
                if first % BLOCK and not scale == old:
                    ratio = old * inverse if scale > 0 else np.float32(0.0)
                    values = plane.astype(np.float32) - np.float32(128.0)
                    again = np.clip(np.rint(values * ratio), -127, 127) if scale > 0 else 0 * values
                    plane[:] = (again + 128).astype(np.uint8)
                slots = self.index[which][first % BLOCK:first % BLOCK + len(new)]
                with np.errstate(invalid="ignore"):
                    q = np.clip(np.rint(new[:, h] * inverse), -127, 127) if scale > 0 else np.zeros_like(new[:, h])
                plane[slots] = (q + 128).astype(np.uint8)
                self.scales[at] = scale

    def values(self, which, table, tokens) -> np.ndarray:
        """[tokens, heads, d] in f32, what the bytes stand for."""
        blocks = -(-tokens // BLOCK)
        out = np.zeros((max(blocks, 1) * BLOCK, self.heads, self.d), np.float32)
        for b in range(blocks):
            plane = self.bytes[table[b], :, which]  # heads, bytes
            u = plane[:, self.index[which]].astype(np.float32) - np.float32(128.0)  # heads, 32, d
            out[b * BLOCK:(b + 1) * BLOCK] = (u * self.scales[table[b], :, which][:, None, None]).transpose(1, 0, 2)
        return out[:tokens]
