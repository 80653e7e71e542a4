"""Routing by logits so large or so far apart that their scores are the same in 64 bits: sigmoids
of 37 and more (1), softmaxes of 746 under the largest (0).  Both scores grow with the
logit, so without a bias, and among experts of one bias, the right order is the
logits' own, the lowest index first among equals: it needs no arithmetic to know."""

from __future__ import annotations

import decimal
import functools

import numpy as np
import pytest

from mote_amd import ops
from test_gpu_experts import route

pytestmark = pytest.mark.gpu

SCORES = [ops.SOFTMAX, ops.SIGMOID]


def weights_of(row, chosen, score, renormalize):
    """In 64 bits; the chosen may be none."""
    x = row.astype(np.float64)
    with np.errstate(over="ignore"):
        if score == ops.SOFTMAX:
            e = np.where(np.isfinite(x), np.exp(np.where(np.isfinite(x), x, 0) - x[np.isfinite(x)].max()), 0)
            s = e / e.sum()
        else:
            s = 1 / (1 + np.exp(-x))
    s = s[chosen]
    return s / s.sum() if renormalize and s.sum() > 0 else s * (not renormalize)


def check(stream, logits, want, score, bias=None, renormalize=True, **groups):
    ids, weights = route(stream, logits, bias, want.shape[1], score, renormalize=renormalize, **groups)
    np.testing.assert_array_equal(ids, want)
    for row, chosen, got in zip(logits, want, weights):
        right = weights_of(row, chosen, score, renormalize)
        # 64 bits throughout and one rounding to 32
        assert (np.abs(got - right) <= 2.0 ** -24 * right + 2.0 ** -148 + 1e-12 * right).all()


def largest_first(logits, top, worth=None):
    """By worth (of the expert's group or bias) and logit, then index."""
    keys = np.zeros_like(logits, np.float64) if worth is None else worth
    return np.array([sorted(range(len(row)), key=lambda e: (-k[e], -float(row[e])))[:top]
                     for row, k in zip(logits, keys)], np.int32)


def far_logits(dtype, tokens, experts):
    """Rows of large, small and equal logits, and of both ends of the type."""
    rng = np.random.default_rng(experts)
    most = float(np.finfo(dtype).max)
    rows = []
    for t in range(tokens):
        low, high = [(38, 60), (-1600, 1600), (746, 3000), (-3000, -746), (29, 31), (-most / 2, most / 2)][t % 6]
        row = rng.uniform(low, high, experts).astype(dtype)
        if t % 3 == 1:
            row[rng.integers(0, experts, experts // 3)] = row[0]
        rows.append(row)
    rows[0][: min(experts, 5)] = [40, 50, 60, 55, 45][: min(experts, 5)]
    if tokens > 1 and experts >= 4:
        rows[1][-4:] = most, -most, most, -most
    return np.array(rows)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("tokens,experts,top", [(1, 5, 3), (6, 8, 8), (13, 64, 6), (12, 100, 64), (9, 256, 8),
                                                (7, 500, 9), (6, 1024, 20)])
def test_far_logits(stream, tokens, experts, top, score, dtype):
    logits = far_logits(dtype, tokens, experts)
    for renormalize in (True, False):
        check(stream, logits, largest_first(logits, top), score, renormalize=renormalize)


def test_underflowed_softmax(stream):
    logits = np.array([[1000, 0, 100, 200, 0]], np.float32)
    check(stream, logits, np.array([[0, 3, 2, 1, 4]], np.int32), ops.SOFTMAX)


def test_zeros_of_both_signs_are_equal(stream):
    logits = np.where(np.arange(96) % 3 == 0, np.float32(0.0), np.float32(-0.0))[None]
    for score in SCORES:
        check(stream, logits, np.arange(7, dtype=np.int32)[None], score)
        check(stream, logits, np.arange(7, dtype=np.int32)[None], score, bias=np.zeros(96))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("experts,top", [(5, 3), (64, 6), (256, 8), (1000, 33)])
def test_far_logits_of_equal_bias(stream, experts, top, score, dtype):
    """Biases that are all the same, or of two sizes further apart than scores can be."""
    logits = far_logits(dtype, 12, experts)
    apart = np.where(np.arange(experts) % 3 == 1, 0.0, -2.0)
    for bias in (np.zeros(experts), np.full(experts, 0.25), apart):
        # (logits of 29 to 31 and scores between: 64 bits tell the 1e-6 between them apart)
        want = largest_first(logits, top, np.broadcast_to(bias, logits.shape))
        check(stream, logits, want, score, bias=bias)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("experts,groups,top_groups,top", [(8, 4, 2, 3), (256, 8, 3, 8), (256, 128, 5, 8),
                                                           (1024, 16, 2, 12), (64, 64, 9, 9)])
def test_far_logits_in_groups(stream, experts, groups, top_groups, top, score):
    """A group's best logit decides, where one choice is its worth; inside the groups, the logits."""
    logits = far_logits(np.float32, 12, experts)
    size = experts // groups
    best = logits.reshape(12, groups, size).max(2)
    kept = np.zeros((12, groups), bool)
    for row, k in zip(best, kept):
        k[sorted(range(groups), key=lambda g: -row[g])[:top_groups]] = True
    want = largest_first(logits, top, np.repeat(kept, size, 1).astype(float))
    check(stream, logits, want, score, groups=groups, top_groups=top_groups, group_best=1)
    if size == 1:
        check(stream, logits, want, score, groups=groups, top_groups=top_groups, group_best=2)


@pytest.mark.parametrize("score", SCORES)
def test_far_logits_inside_groups_of_two_best(stream, score):
    """The two best of groups whose worths are apart; the logits decide inside them."""
    logits = np.full((1, 64), -30.0, np.float32)
    logits[0, 16:32] = 40 + np.arange(16) % 7
    logits[0, 48:] = 60 - np.arange(16) % 5 if score == ops.SIGMOID else 1000 - np.arange(16)
    kept = np.repeat([[0, 1, 0, 1]], 16, 1).astype(float)
    for bias in (None, np.zeros(64)):
        check(stream, logits, largest_first(logits, 24, kept), score, bias=bias, groups=4, top_groups=2, group_best=2)


DIGITS = decimal.Context(prec=700, Emin=-(10 ** 6), Emax=10 ** 6)


@functools.lru_cache(maxsize=None)
def exact_exp(x):
    return decimal.Decimal(x).exp(DIGITS)


def exact_worths(row, groups, score):
    """Sums of each group's two best scores, to 700 digits (a softmax's without the row's sum)."""
    with decimal.localcontext(DIGITS):
        e = [exact_exp(float(x)) for x in row]
        s = e if score == ops.SOFTMAX else [v / (1 + v) for v in e]
        size = len(row) // groups
        return [sum(sorted(s[g * size: (g + 1) * size])[-2:]) for g in range(groups)]


@pytest.mark.parametrize("bias", [None, 0.0, 0.25])
@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("experts,groups,top_groups,top", [(16, 4, 2, 5), (256, 8, 3, 8), (256, 128, 40, 20)])
def test_far_groups_of_two_best(stream, experts, groups, top_groups, top, score, bias):
    """Worths that 64 bits hold as 2, 1 or 0 alike: sums of two sigmoids of 40 to 600, of one of those and
    one of -600 to -40, and of two such; softmaxes of logits thousands apart."""
    rng = np.random.default_rng(experts)
    size = experts // groups
    rows = []
    for kind in range(6):
        row = rng.uniform(40, 600, (groups, size)) * np.where(rng.random((groups, size)) < 0.5, 1, -1)
        if kind == 0:
            row = np.abs(row)
        elif kind == 1:
            row = -np.abs(row)
        elif kind == 2:  # one large logit in each group
            row = -np.abs(row)
            row[np.arange(groups), rng.integers(0, size, groups)] *= -1
        elif kind == 3:  # sums of exactly 1, and others next to it
            row = -np.abs(row) - 1
            row[:, 0] = rng.integers(40, 300, groups)
            row[:, -1] = -row[:, 0] + rng.integers(-1, 2, groups)
        elif kind == 4:  # few sizes: equal groups among others
            row = np.round(row / 200) * 200
        else:  # all small but one group
            row = -np.abs(row)
            row[-1] += 1200 if score == ops.SOFTMAX else 0
        rows.append(row.reshape(-1))
    logits = np.array(rows).astype(np.float32)
    kept = np.zeros((len(rows), groups))
    for row, k in zip(logits, kept):
        worth = exact_worths(row, groups, score)
        k[sorted(range(groups), key=lambda g: worth[g], reverse=True)[:top_groups]] = 1  # (a sign change would round)
    want = largest_first(logits, top, np.repeat(kept, size, 1))
    check(stream, logits, want, score, bias=None if bias is None else np.full(experts, bias), groups=groups,
          top_groups=top_groups, group_best=2)


@pytest.mark.parametrize("bias", [None, 0.0])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("top_groups", [2, 4, 6, 9])
def test_softmax_groups_of_any_size(stream, top_groups, dtype, bias):
    """Groups of two best that all underflow, down to the type's lowest value: their best logits lie more
    than log 2 apart, so they and then the second ones decide."""
    rng = np.random.default_rng(top_groups)
    lowest = float(np.finfo(dtype).min)
    far = [-2000, -2001, -5000.5, -30000, lowest / 2, lowest]
    if dtype == np.float32:
        far += [-1e5, -1e7, -3e9, -1e15, -2.0 ** 60, -1e20, -1e30]
    logits = np.empty((40, 16, 4), dtype)
    for row in logits:
        best = rng.choice(far, 16).astype(dtype)
        row[:] = lowest
        row[np.arange(16), rng.integers(0, 4, 16)] = best
        row[rng.integers(0, 16)] = 0
    ordered = np.sort(logits.astype(np.float64), 2)[:, :, ::-1]
    kept = np.zeros((40, 16))
    for row, k in zip(ordered, kept):
        k[sorted(range(16), key=lambda g: (-row[g, 0], -row[g, 1]))[:top_groups]] = 1
    logits = logits.reshape(40, 64)
    want = largest_first(logits, 7, np.repeat(kept, 4, 1))
    check(stream, logits, want, ops.SOFTMAX, bias=None if bias is None else np.zeros(64), groups=16,
          top_groups=top_groups, group_best=2)
