"""Microscaled rows, routing and the experts' products in 64 bits, from their
definitions (include/mote_hip.h), on the host."""

from __future__ import annotations

import math

import numpy as np

BLOCK, PADDED = 32, 128
UP = {4: np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6]),
      6: np.concatenate([np.arange(16) / 8, 2 + np.arange(8) / 4, 4 + np.arange(8) / 2])}


def padded(features):
    return -(-features // PADDED) * PADDED


def elements(bits):
    """What each code stands for."""
    return np.concatenate([UP[bits], -UP[bits]])


def pack(codes, bits):
    """Codes [rows, padded] to values [rows, padded bits / 8]."""
    rows, width = codes.shape
    bit = (codes[..., None].astype(np.uint8) >> np.arange(bits, dtype=np.uint8)) & 1
    stream = np.packbits(bit.reshape(rows, width // BLOCK, BLOCK * bits), axis=2, bitorder="little")
    blocks = width // BLOCK
    return np.concatenate([stream[:, :, :16].reshape(rows, 16 * blocks),
                           stream[:, :, 16:].reshape(rows, (4 * bits - 16) * blocks)], 1)


def unpack(values, bits):
    rows, blocks = values.shape[0], values.shape[1] // (4 * bits)
    stream = np.concatenate([values[:, : 16 * blocks].reshape(rows, blocks, 16),
                             values[:, 16 * blocks:].reshape(rows, blocks, 4 * bits - 16)], 2)
    bit = np.unpackbits(stream, axis=2, bitorder="little").reshape(rows, blocks * BLOCK, bits)
    return (bit.astype(np.int64) << np.arange(bits)).sum(2)


def read(values, scales, bits):
    """What rows stand for, padding included."""
    with np.errstate(invalid="ignore"):
        of = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return elements(bits)[unpack(values, bits)] * np.repeat(of, BLOCK, axis=1)


def quantize(x, bits):
    """Values and scales of rows x [rows, features]."""
    rows, features = x.shape
    x = np.asarray(x, np.float64).reshape(rows, -1, BLOCK)
    most = np.abs(x).max(2)
    bad = ~np.isfinite(most)
    mantissa, exponent = np.frexp(np.where(bad, 1.0, most))
    shared = np.where(most > 0, exponent - 1 - 2, -127).clip(-127)
    y = np.where(bad[..., None], 0.0, x) / 2.0 ** shared[..., None]
    up = UP[bits]
    size = np.minimum(np.abs(y), up[-1])
    above = np.searchsorted(up, size).clip(1, len(up) - 1)
    low, high = up[above - 1], up[above]
    code = np.where((high - size < size - low) | ((high - size == size - low) & (above % 2 == 0)), above, above - 1)
    code = code | np.where(np.signbit(y) & ~bad[..., None], len(up), 0)
    out = np.zeros((rows, padded(features)), np.int64)
    out[:, :features] = code.reshape(rows, features)
    scales = np.zeros((rows, padded(features) // BLOCK), np.uint8)
    scales[:, : features // BLOCK] = np.where(bad, 255, shared + 127)
    return pack(out, bits), scales


def random_rows(rng, rows, features, bits, low=124, high=131):
    """Random codes with scale bytes low .. high - 1, zeros in the padding."""
    codes = np.zeros((rows, padded(features)), np.int64)
    codes[:, :features] = rng.integers(0, 1 << bits, (rows, features))
    scales = np.zeros((rows, padded(features) // BLOCK), np.uint8)
    scales[:, : features // BLOCK] = rng.integers(low, high, (rows, features // BLOCK))
    return pack(codes, bits), scales


def route(logits, bias, top, score, groups=1, top_groups=1, best=2, renormalize=True, scale=1.0):
    """ids and weights, one expert after the other."""
    x = np.asarray(logits, np.float64)
    tokens, experts = x.shape
    ids, weights = np.full((tokens, top), -1, np.int32), np.zeros((tokens, top))
    of = np.arange(experts) // (experts // groups)
    for t, row in enumerate(x):
        there = np.isfinite(row)
        if not there.any():
            continue
        with np.errstate(over="ignore", invalid="ignore"):
            if score == 0:
                s = np.where(there, np.exp(np.where(there, row, 0) - row[there].max()), 0)
                s = s / math.fsum(s)
            else:
                s = 1 / (1 + np.exp(-row))
            c = s + (0 if bias is None else np.asarray(bias, np.float64))
        there &= np.isfinite(c)
        if top_groups < groups:
            worth = []
            for g in range(groups):
                mine = np.sort(c[there & (of == g)])[::-1][:best]
                worth.append(mine.sum() if mine.size else -np.inf)
            order = sorted(range(groups), key=lambda g: -worth[g])[:top_groups]
            there &= np.isin(of, order)
        order = sorted(np.flatnonzero(there), key=lambda e: -c[e])[:top]  # the lowest first among equals
        ids[t, : len(order)] = order
        weights[t, : len(order)] = s[order]
        if renormalize:
            total = weights[t].sum()
            weights[t] = weights[t] / total if total > 0 else 0
    return ids, weights * scale


def plan(ids, experts):
    flat = np.asarray(ids).reshape(-1)
    rows = [p for e in range(experts) for p in np.flatnonzero(flat == e)]
    offsets = np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(experts)])]).astype(np.int32)
    return offsets, np.array(rows + [-1] * (flat.size - len(rows)), np.int32)


def gate_up(x, w, offsets, rows, top):
    """x [tokens, K], w [experts, 2 I, K] in 64 bits: silu(gate) up, gate and up
    of each row of the plan in use."""
    inner = w.shape[1] // 2
    out = np.zeros((offsets[-1], 2 * inner))
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        out[a:b] = x[rows[a:b] // top] @ w[e].T
    gate, up = out[:, :inner], out[:, inner:]
    with np.errstate(over="ignore"):
        return gate / (1 + np.exp(-gate)) * up, gate, up


def down(h, w, ids, offsets, rows, weights):
    """The weighted sums, and of their terms' sizes."""
    tokens, top = ids.shape
    y, size = np.zeros((tokens, w.shape[1])), np.zeros((tokens, w.shape[1]))
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        for i in range(a, b):
            t, j = divmod(int(rows[i]), top)
            term = weights[t, j] * (h[i] @ w[e].T)
            y[t] += term
            size[t] += np.abs(term)
    return y, size
