"""The CPU restatement of the operators around a prompt chunk's layers (oracle/prompt.py) against closed forms:
attention over equal rows, norms of known heads, codes at half-way points, counters by hand, softmax of few logits."""
import math

import numpy as np
import pytest

from oracle import draft, prompt


def test_features_round_to_eleven_bits():
    rows = np.zeros((40, 656), np.uint8)
    rows[:, 640:656] = np.asarray([1, 1, 1, 1], "<f4").view(np.uint8)
    rows[0, 640:644] = np.asarray([1 + 2.0 ** -11 + 2.0 ** -20], "<f4").view(np.uint8)  # rounds up
    rows[1, 640:644] = np.asarray([1 + 2.0 ** -11], "<f4").view(np.uint8)               # halves to the even step
    rows[:, :512] = draft.e4m3_bytes(np.ones((40, 512), np.float32))
    rows[35, 640:644] = np.asarray([3e38], "<f4").view(np.uint8)  # its tile's rows keep exponents of their own
    rows[36, 0:1] = draft.e4m3_bytes(np.asarray([2.0 ** -9], np.float32))
    rows[3, 640:656] = np.asarray([2.0 ** -9] * 4, "<f4").view(np.uint8)  # one exponent
    rows[3, 0:1] = draft.e4m3_bytes(np.asarray([2.0 ** -9], np.float32))
    rows[3, 512:514] = np.asarray([0x3F81], "<u2").view(np.uint8)  # bf16 1 + 2^-7
    key, value, odd = prompt.features(rows)
    assert value[0, 0] == 1 + 2.0 ** -10 and value[1, 0] == 1.0 and value[2, 0] == 1.0 and not odd.any()
    assert abs(value[35, 0] / 3e38 - 1) <= 2.0 ** -11 and value[36, 0] == 2.0 ** -9 and value[36, 200] == 1.0
    assert value[3, 0] == 2.0 ** -18 and value[3, 1] == 2.0 ** -9 and key[3, 512] == 1 + 2.0 ** -7
    assert np.array_equal(key[:, :512], value) and np.array_equal(prompt.features(rows[:32])[1], value[:32])


def test_attention_over_equal_logits_is_the_mean():
    rows = np.zeros((3, 656), np.uint8)
    rows[:, :512] = draft.e4m3_bytes(np.repeat([[1.0], [2.0], [6.0]], 512, axis=1).astype(np.float32))
    rows[:, 640:656] = np.asarray([1, 2, 3, 4], "<f4").view(np.uint8)
    key, value, odd = prompt.features(rows)
    assert not odd.any() and value[2, 200] == 12.0 and key.shape == (3, 576)
    out, lse, bound, slip = prompt.attention(np.zeros((2, 576)), key, value, 0.1)
    assert np.allclose(out[0, ::128], 3.0 * np.asarray([1, 2, 3, 4])) and np.allclose(lse, math.log(3))
    assert np.all(bound > 0) and np.all(slip > 0)
    out, lse, _, _ = prompt.attention(np.ones((2, 576)), key[:0], value[:0], 0.1)
    assert not out.any() and np.all(lse == -np.inf)
    rows[1, 640:644] = np.asarray([np.inf], "<f4").view(np.uint8)
    assert prompt.features(rows)[2].tolist() == [False, True, False]


@pytest.mark.parametrize("kind", ["rms", "layer", None])
def test_norms(kind):
    x = np.asarray([[3.0, -1.0, 3.0, -1.0], [0.0, 0.0, 0.0, 0.0]])
    y, bound = prompt.normed(x, kind, weight=[1, 2, 3, 4], bias=[0, 0, 0, 1], epsilon=1e-30)
    want = {"rms": np.asarray([3, -2, 9, -4]) / math.sqrt(5) + [0, 0, 0, 1], "layer": [1, -2, 3, -3], None: [3, -2, 9, -3]}[kind]
    assert np.allclose(y[0], want) and np.array_equal(y[1], [0, 0, 0, 1]) and np.all(bound >= 0)


def test_codes_round_to_even_steps():
    y = np.zeros((1, 128))
    y[0, :5] = [448.0, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10]  # steps of 2 above 16, of 2^-9 below 2^-6
    values, scale = prompt.codes(y)
    assert scale[0] == 1.0 and values[0, :5].tolist() == [448.0, 16.0, 20.0, 0.0, 2.0 ** -8]
    assert prompt.codes(np.zeros((2, 128)))[1].tolist() == [1.0, 1.0]


def test_history_by_hand():
    h = prompt.History(2, 40)
    h.load(1, [3, 3, 39, 5, 40, -1, 5], 3)
    h.append(1, [5, 7])
    counts, seen = h.arrays()
    assert counts[1, 5] == 3 and counts[1, 7] == 1 and counts[1, 3] == 0 and counts.sum() == 4
    assert seen.view(np.uint32)[1].tolist() == [1 << 3 | 1 << 5 | 1 << 7, 1 << 7] and not seen[0].any()


def test_logits_and_probabilities():
    x, bound, odd = prompt.logits([2.0, -2.0, 1.0, 0.5], wrote={0: 2}, has={0, 1}, way=[2], repetition=2.0, presence=0.25,
                                  frequency=0.5, biases=[(3, 1.0), (3, 0.5), (-1, 9.0)], allowed=np.asarray([True, True, True, False]))
    assert x[:3].tolist() == [1.0 - 0.25 - 1.0, -4.0, 0.5 - 0.25 - 0.5] and x[3] == -np.inf and not odd
    p, _ = prompt.probabilities(np.asarray([0.0, math.log(3.0), -np.inf]), np.zeros(3), 1.0)
    assert np.allclose(p, [0.25, 0.75, 0.0])
    assert prompt.probabilities(np.asarray([1.0, 5.0, 5.0]), np.zeros(3), 0.0)[0].tolist() == [0, 1, 0]
    assert prompt.probabilities(np.asarray([np.inf, 5.0, np.inf]), np.zeros(3), 1.0)[0].tolist() == [0.5, 0, 0.5]
    assert not prompt.probabilities(np.full(3, -np.inf), np.zeros(3), 1.0)[0].any()
    assert prompt.logits([np.nan, 1.0])[2] and not prompt.logits([np.nan, 1.0], allowed=np.asarray([False, True]))[2]
