"""CPU restatement in 64 bits of the operators on either side of a prompt chunk's layers
(include/kvip_hip_prompt.h). TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).

features         - keys and values of cached rows as chunk attention takes them (rounded once to fp16 under an exponent)
attention        - softmax attention of one token, with a bound for the kernel's roundings
normed           - norm, weight and bias of heads, with a bound
turned           - oracle.draft's turn, with a bound
codes            - e4m3 values and scales of heads
History          - what requests hold, as plain counters
logits           - the adjusted logits of a row, with a bound
probabilities    - softmax or first largest, with a bound
Pinned in tests/test_oracle_prompt.py by closed forms.
"""
from __future__ import annotations

from collections import Counter

import numpy as np

from oracle import draft

BLOCK = 128
FP32 = 2.0 ** -24  # half a step of 32 bits, of the value; so FP16 below
FP16 = 2.0 ** -11


def features(rows, positions=None):
    """rows uint8 [n, >= 656] of one request, at positions 0, 1, ... or as given -> (key [n, 576], value [n, 512], odd [n]: a
    value is no finite number). Products in 32 bits, rounded to fp16 under the exponent that takes the largest finite
    feature of the 32 positions' rows (those that are odd left out) to 2^11 .. 2^15 (a multiple of 4), or, where the rows'
    own exponents differ by more than 12, each under its own."""
    positions = np.arange(len(rows)) if positions is None else np.asarray(positions)
    with np.errstate(over="ignore", invalid="ignore"):
        nope, rope, scales = draft.row_parts(rows)
        product = nope.astype(np.float32) * np.repeat(scales.astype(np.float32), 128, axis=1)
        odd = ~np.isfinite(product).all(1)
        product[odd] = 0
        key = np.concatenate([product, rope.astype(np.float32)], axis=1)
        for tile in np.unique(positions // 32):
            at = np.flatnonzero(positions // 32 == tile)
            sizes = np.abs(np.where(np.isfinite(key[at]), key[at], 0)).max(1)
            exponents = -(-(np.where(sizes >= 2.0 ** -126, np.frexp(sizes)[1] - 1, -127) - 14) // 4) * 4
            if np.any(sizes > 0) and exponents.max() - exponents[sizes > 0].min() <= 12:
                exponents[:] = exponents.max()
            for i, exponent in zip(at, exponents):
                key[i] = np.ldexp(np.ldexp(key[i].astype(np.float64), -exponent).astype(np.float16).astype(np.float64), exponent)
    return key.astype(np.float64), key[:, :512].astype(np.float64), odd


def attention(query, key, value, scale):
    """query [heads, 576] of one token over the rows it sees. Returns (output [heads, 512], lse [heads], bound
    [heads, 512], lse bound [heads]): the bounds hold for probabilities rounded to fp16 (2^-11; the smallest, of tiles whose
    exponent is 4 below others', 2^-31 of the maximum's), dot products of 576 terms, exponentials and sums of n
    terms in 32 bits."""
    q, n = np.asarray(query, np.float64), len(key)
    if n == 0:
        zero = np.zeros((len(q), value.shape[1]))
        return zero, np.full(len(q), -np.inf), zero, np.zeros(len(q))
    logits = scale * (q @ key.T)
    top = logits.max(1, keepdims=True)
    p = np.exp(logits - top)
    whole = p.sum(1, keepdims=True)
    p /= whole
    slip = abs(scale) * (np.abs(q) @ np.abs(key).T).max(1) * (576 + 8) * FP32 + np.abs(logits).max(1) * 8 * FP32
    sums = n * 2 * FP32 + 16 * FP32
    bound = (p @ np.abs(value)) * (FP16 + 2 * slip + sums)[:, None] + 2.0 ** -31 * np.abs(value).sum(0) / whole
    return p @ value, top[:, 0] + np.log(whole[:, 0]), bound, slip + sums + np.abs(top[:, 0]) * 4 * FP32


def normed(x, kind, weight=None, bias=None, epsilon=1e-6):
    """x [..., dim] normed ("rms", "layer" or None), times weight, plus bias; and a bound for the same in 32 bits:
    sums of dim terms, a difference, a square root, a quotient, two products and a sum."""
    x = np.asarray(x, np.float64)
    dim = x.shape[-1]
    size = np.abs(x).mean(-1, keepdims=True)
    y, off = x, np.zeros_like(x)
    if kind == "layer":
        y = x - x.mean(-1, keepdims=True)
        off = FP32 * ((dim + 2) * size + 2 * np.abs(x))
    factor = np.ones_like(size)
    if kind is not None:
        square = (y * y).mean(-1, keepdims=True) + epsilon
        factor = 1 / np.sqrt(square)
        # The mean square's own error, halved by the root: from the differences' errors and from the sum.
        off = off * factor + np.abs(y) * factor * ((off * np.abs(y)).mean(-1, keepdims=True) / square + (dim / 2 + 8) * FP32)
    y = y * factor
    w = np.ones(dim) if weight is None else np.asarray(weight, np.float64)
    b = np.zeros(dim) if bias is None else np.asarray(bias, np.float64)
    return y * w + b, off * np.abs(w) + 4 * FP32 * (np.abs(y * w) + np.abs(b))


def turned(y, off, positions, frequencies, half, magnitude):
    """The turn of values y that are off by up to `off`: an angle off by 2 pi 2^-25, sine and cosine by 2 units of
    2^-24, three products and sums."""
    out = draft.turned(y, positions, frequencies, half, magnitude)
    pairs = len(frequencies)
    first, second = (slice(0, pairs), slice(pairs, 2 * pairs)) if half else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
    bound = np.array(off)
    sums = (np.abs(y[..., first]) + np.abs(y[..., second])) * 16 * FP32 + (off[..., first] + off[..., second]) * 1.001
    bound[..., first] = bound[..., second] = sums * magnitude
    return out, bound


def codes(y):
    """(values that the e4m3 codes of heads y [..., 128] stand for, under their scale; the scale)."""
    y = np.asarray(y, np.float64)
    largest = np.fmax.reduce(np.abs(y), axis=-1) / 448
    scale = np.where(largest > 0, largest, 1.0)
    x = y / scale[..., None]
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))), -6) - 3)
    return np.round(x / step) * step, scale


class History:
    """What each of `batch` requests holds: how often it wrote a token, and which it has at all."""

    def __init__(self, batch, vocab):
        self.vocab, self.wrote, self.has = vocab, [Counter() for _ in range(batch)], [set() for _ in range(batch)]

    def load(self, request, tokens, prompt):
        tokens = [int(t) for t in tokens]
        good = [0 <= t < self.vocab for t in tokens]
        self.wrote[request] = Counter(t for i, (t, ok) in enumerate(zip(tokens, good)) if ok and i >= prompt)
        self.has[request] = {t for t, ok in zip(tokens, good) if ok}

    def append(self, request, tokens):
        good = [int(t) for t in tokens if 0 <= t < self.vocab]
        self.wrote[request].update(good)
        self.has[request].update(good)

    def arrays(self):
        """(counts [batch, vocab], seen words int32 [batch, (vocab + 31) / 32])."""
        counts = np.zeros((len(self.wrote), self.vocab), np.int32)
        seen = np.zeros((len(self.wrote), -(-self.vocab // 32)), np.uint32)
        for b, (wrote, has) in enumerate(zip(self.wrote, self.has)):
            for t, n in wrote.items():
                counts[b, t] = n
            for t in has:
                seen[b, t // 32] |= np.uint32(1 << t % 32)
        return counts, seen.view(np.int32)


def logits(x, *, wrote=None, has=None, way=(), repetition=1.0, presence=0.0, frequency=0.0, biases=(), allowed=None):
    """Adjusted logits of one row: wrote and has (of a History), the drafted tokens on the way to the row, biases as
    (token, value) pairs in order, allowed as bool [vocab]. Returns (x, bound, odd): the bound for the same in 32
    bits, odd where an allowed x is a NaN."""
    x = np.array(x, np.float64)
    vocab = len(x)
    n = np.zeros(vocab)
    for t, count in (wrote or {}).items():
        n[t] += count
    held = np.zeros(vocab, bool)
    held[list(has or ())] = True
    for t in way:
        if 0 <= t < vocab:
            n[t] += 1
            held[t] = True
    with np.errstate(invalid="ignore"):
        x = np.where(held, np.where(x > 0, x / repetition, x * repetition), x)
        size = np.abs(x) + (n > 0) * (abs(presence) + abs(frequency) * n)
        x = x - (n > 0) * (presence + frequency * n)
        for t, value in biases:
            if 0 <= t < vocab:
                x[t] += value
                size[t] += abs(value)
        bound = np.where(np.isfinite(size), size, 0.0) * (4 + len(biases)) * FP32 * (held | (size != np.abs(x)))
    if allowed is not None:
        x = np.where(allowed, x, -np.inf)
    odd = np.isnan(x)
    return np.where(odd, -np.inf, x), bound, bool(odd.any())


def probabilities(x, bound, temperature=1.0):
    """(probabilities, bound) of adjusted logits that are off by up to `bound`; temperature not above 0: one place."""
    if x.max() == -np.inf:
        return np.zeros_like(x), np.zeros_like(x)
    if not temperature > 0:
        p = np.zeros_like(x)
        p[int(np.argmax(x))] = 1.0
        return p, np.zeros_like(x)
    if x.max() == np.inf:
        p = (x == np.inf) / np.count_nonzero(x == np.inf)
        return p, p * 4 * FP32
    away = np.where(x == -np.inf, 0.0, x - x.max())
    weight = np.where(x == -np.inf, 0.0, np.exp(away / temperature))
    p = weight / weight.sum()
    off = (bound + bound.max() + np.abs(away) * 4 * FP32) / temperature + 8 * FP32
    # The sum: the terms' own errors, weighted by them, and of runs of up to 2^17 terms some 600 sums one after another.
    return p, p * (off + (p * off).sum() + 1024 * FP32) * 1.01 + 2.0 ** -126
