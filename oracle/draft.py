"""CPU restatement in 64 bits of the operators of a drafted round (include/kvip_hip_draft.h). TEST
INFRASTRUCTURE ONLY (see oracle/__init__.py).

turned            - rotary positions, by complex numbers
e4m3_bytes        - fp32 values to fp8 e4m3 bytes, halves to the even code
stored_rows       - the 656-byte rows of latents (scales and codes exactly as stated)
row_parts         - features, rope and scales of rows in 64 bits
tree_attention    - softmax attention of step tokens, with a bound for the kernel's roundings
ancestors         - visibility and depth of a tree's tokens
Tables            - page tables as plain lists
verify            - the walk and the drawn token
Pinned in tests/test_oracle_draft.py by closed forms and, for verify, by the distribution of its tokens.
"""
from __future__ import annotations

import math

import numpy as np

from oracle.indexer import fp8_e4m3_decode

BLOCK = 128
ROW = 656


def turned(x, positions, frequencies, half, magnitude=1.0, inverse=False):
    """x [tokens, ..., dim] with its first 2 len(frequencies) features turned."""
    y = np.array(x, np.float64)
    pairs = len(frequencies)
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(frequencies, np.float64)
    turn = magnitude * np.exp(1j * (-angle if inverse else angle))
    turn = turn.reshape((len(y),) + (1,) * (y.ndim - 2) + (pairs,))
    first, second = (slice(0, pairs), slice(pairs, 2 * pairs)) if half else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
    z = (y[..., first] + 1j * y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


_CODES = np.asarray([fp8_e4m3_decode(np.asarray([c], np.uint8))[0] for c in range(127)], np.float64)  # 0 .. 448


def e4m3_bytes(values):
    """float32 within +-448 or NaN -> e4m3 bytes, to the nearest code, halves to the even one."""
    x = np.abs(np.asarray(values, np.float64))
    hi = np.clip(np.searchsorted(_CODES, x), 1, 126)
    lo = hi - 1
    below, above = x - _CODES[lo], _CODES[hi] - x
    code = np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return (np.where(np.isnan(x), 127, code) | (np.signbit(values) * 128)).astype(np.uint8)


def stored_rows(latent):
    """(codes uint8 [n, 512], scales float32 [n, 4]) of latents [n, 512]."""
    x = np.asarray(latent, np.float32).reshape(-1, 4, 128)
    scales = np.fmax.reduce(np.abs(x), axis=2) / np.float32(448)  # of the numbers among them
    scales = np.where(scales > 0, scales, np.float32(1)).astype(np.float32)
    with np.errstate(invalid="ignore"):  # an infinity over its own scale
        return e4m3_bytes(np.clip(x / scales[:, :, None], -448, 448)).reshape(-1, 512), scales


def row_parts(rows):
    """rows uint8 [n, >= 656] -> (nope [n, 512], rope [n, 64], scales [n, 4]) in 64 bits."""
    rows = np.ascontiguousarray(np.asarray(rows, np.uint8)[:, :ROW])
    rope = (rows[:, 512:640].copy().view("<u2").astype(np.uint32) << 16).view(np.float32)
    return (fp8_e4m3_decode(rows[:, :512]).astype(np.float64), rope.astype(np.float64),
            rows[:, 640:656].copy().view("<f4").astype(np.float64))


def tree_attention(query, rows, sees, scale):
    """query [heads, 576] of one token, rows uint8 [n, >= 656], sees bool [n]. Returns (output [heads, 512],
    lse [heads], bound [heads, 512], lse bound [heads]): the bounds hold for probabilities times scales rounded to
    bf16 (2^-8), dot products of 576 terms, exponentials and sums of n terms in 32 bits (2^-24 each)."""
    q = np.asarray(query, np.float64)
    nope, rope, scales = row_parts(rows[np.flatnonzero(sees)])
    value = nope * np.repeat(scales, 128, axis=1)
    key = np.concatenate([value, rope], axis=1)
    n = len(key)
    if n == 0:
        zero = np.zeros((len(q), 512))
        return zero, np.full(len(q), -np.inf), zero, np.zeros(len(q))
    logits = scale * (q @ key.T)
    top = logits.max(1, keepdims=True)
    p = np.exp(logits - top)
    whole = p.sum(1, keepdims=True)
    p /= whole
    slip = abs(scale) * (np.abs(q) @ np.abs(key).T).max(1) * (576 + 8) * 2.0 ** -24 + np.abs(logits).max(1) * 2.0 ** -21
    sums = n * 2.0 ** -23 + 2.0 ** -20
    spread = (p @ np.abs(value)) * (2.0 ** -8 + 2 * slip + sums)[:, None]
    return p @ value, top[:, 0] + np.log(whole[:, 0]), spread, slip + sums + np.abs(top[:, 0]) * 2.0 ** -22


def ancestors(parents):
    """(visibility bits, depth) of a request's tokens; parents before children."""
    bits, depth = [], []
    for i, up in enumerate(parents):
        ok = 0 <= up < i
        bits.append(1 << i | (bits[up] if ok else 0))
        depth.append(depth[up] + 1 if ok else 0)
    return bits, depth


class Tables:
    """Page tables as plain lists: pages[b], lengths[b], the stack of free pages."""

    def __init__(self, batch, max_blocks, num_blocks, max_tokens):
        self.pages = [[] for _ in range(batch)]
        self.lengths, self.bases, self.steps = [0] * batch, [0] * batch, [0] * batch
        self.stack = list(range(num_blocks - 1, -1, -1))
        self.max_blocks, self.max_tokens = max_blocks, max_tokens

    def extend(self, counts, parents=None):
        """(cu_seqlens, slots, positions, visible, status)."""
        status, rows, wanted = 0, 0, 0
        cu, slots, positions, visible = [0], [-1] * self.max_tokens, [0] * self.max_tokens, [0] * self.max_tokens
        have = len(self.stack)
        for b, count in enumerate(counts):
            n, base = max(count, 0), self.lengths[b]
            fits = count >= 0 and base + n <= self.max_blocks * BLOCK and rows + n <= self.max_tokens and \
                (parents is None or n <= 64)
            status |= 0 if fits else 16
            step = n if fits else 0
            need = -(-(base + step) // BLOCK) - len(self.pages[b])
            wanted += need
            if need and wanted > have:
                status |= 8
                step = 0
            else:
                self.pages[b] += [self.stack.pop() for _ in range(need)]
            self.bases[b], self.steps[b], self.lengths[b] = base, step, base + step
            there = min(n, max(self.max_tokens - rows, 0))
            tree = None if parents is None else [int(x) for x in parents[rows:rows + min(there, 64)]]
            if tree is not None:
                status |= 32 if any(not -1 <= up < i for i, up in enumerate(tree)) else 0
                bits, depth = ancestors(tree)
            for i in range(there):
                if tree is not None and i >= 64:
                    continue
                positions[rows + i] = base + (i if tree is None else depth[i])
                visible[rows + i] = (1 << min(i + 1, 64)) - 1 if tree is None else bits[i]
                if step:
                    slots[rows + i] = self.pages[b][(base + i) // BLOCK] * BLOCK + (base + i) % BLOCK
            rows += n
            cu.append(min(rows, self.max_tokens))
        return cu, slots, positions, visible, status

    def truncate(self, lengths):
        freed = []
        for b, length in enumerate(lengths):
            length = min(max(length, 0), self.lengths[b])
            keep = -(-length // BLOCK)
            freed += self.pages[b][keep:]
            del self.pages[b][keep:]
            self.lengths[b] = self.bases[b] = length
            self.steps[b] = 0
        self.stack += freed[::-1]

    def commit(self, kept):
        self.truncate([base + min(max(k, 0), step) for base, k, step in zip(self.bases, kept, self.steps)])


def verify(probs, tokens, parents, draft, uniforms, final):
    """One request: probs [n, vocab], tokens [n], parents [n] or None, draft [n, vocab] or None. Returns (path, out tokens),
    the last out token -1 where none can be drawn."""
    n, vocab = probs.shape
    probs = np.asarray(probs, np.float64)
    up = list(range(-1, n - 1)) if parents is None else [int(x) if 0 <= x < i else -1 for i, x in enumerate(parents)]
    named = [0 <= int(t) < vocab for t in tokens]

    def weight(table, row, i):
        x = float(table[row, int(tokens[i])])
        return x if x > 0 else 0.0

    at, path = 0, [0]
    while True:
        children = [i for i in range(at + 1, n) if up[i] == at and named[i]]
        u, taken, weighty = float(uniforms[at]), None, -1
        if draft is not None:
            if children and u * float(draft[at, int(tokens[at + 1])]) < weight(probs, at, at + 1):
                taken = at + 1
        else:
            low, seen = 0.0, set()
            for i in children:
                if int(tokens[i]) in seen:
                    continue
                seen.add(int(tokens[i]))
                high = low + weight(probs, at, i)
                if low <= u < high:
                    taken = i
                    break
                weighty = int(tokens[i]) if weight(probs, at, i) > 0 else weighty
                low = high
        if taken is None:
            break
        at = taken
        path.append(at)
    rest = probs[at].copy()
    if draft is not None:
        if at + 1 < n:
            rest = rest - np.asarray(draft[at], np.float64)
    else:
        rest[[int(tokens[i]) for i in children]] = 0.0
    rest = np.where(rest > 0, rest, 0.0)
    whole = rest.sum()
    if whole == 0 and draft is not None:  # a target that is nowhere above its draft
        rest = np.where(probs[at] > 0, probs[at], 0.0)
        whole = rest.sum()
    last = weighty if whole == 0 else -1  # children that are the whole target
    if 0 < whole < math.inf:
        passed = np.flatnonzero((np.cumsum(rest) > float(final) * whole) & (rest > 0))
        last = int(passed[0]) if len(passed) else int(np.flatnonzero(rest)[-1])
    return path, [int(tokens[i]) for i in path[1:]] + [last]
