"""The CPU restatement of the drafted round (oracle/draft.py) against closed forms: turns by known angles,
every e4m3 code and half-way point, attention with equal logits, ancestors by hand, and for the
verification the distribution of its first token over all drafts and uniforms, which has to be the target's."""
import math

import numpy as np
import pytest

from kvip_amd.operators.rotary import rotary_frequencies
from oracle import draft
from oracle.indexer import fp8_e4m3_decode


@pytest.mark.parametrize("half", [False, True])
def test_turn_by_a_quarter_and_back(half):
    x = np.arange(12, dtype=np.float64).reshape(2, 6)
    y = draft.turned(x, [1, 0], [math.pi / 2, 0.0], half, magnitude=2.0)
    first, second = (slice(0, 2), slice(2, 4)) if half else (slice(0, 4, 2), slice(1, 4, 2))
    assert np.allclose(y[0, first], 2 * np.asarray([-x[0, second][0], x[0, first][1]]))
    assert np.allclose(y[1, :4], 2 * x[1, :4]) and np.array_equal(y[:, 4:], x[:, 4:])
    back = draft.turned(y, [1, 0], [math.pi / 2, 0.0], half, magnitude=0.5, inverse=True)
    assert np.allclose(back, x)


def test_frequencies():
    plain, one = rotary_frequencies(64)
    assert one == 1.0 and plain[0] == 1.0 and math.isclose(plain[16], 0.01)
    assert rotary_frequencies(64, scaling={"kind": "linear", "factor": 4.0})[0] == [f / 4.0 for f in plain]
    ntk = rotary_frequencies(64, scaling={"kind": "ntk", "factor": 8.0})[0]
    assert ntk[0] == 1.0 and math.isclose(ntk[31], plain[31] / 8.0)  # the slowest pair is stretched by the factor
    yarn, magnitude = rotary_frequencies(64, scaling={"kind": "yarn", "factor": 40.0, "original": 4096})
    turns = [4096 * f / (2 * math.pi) for f in plain]
    for f, g, t in zip(plain, yarn, turns):
        assert f / 40.0 * (1 - 1e-12) <= g <= f
        assert g == f or t < 48  # fast pairs stay (the limits are rounded outwards by one pair)
        assert math.isclose(g, f / 40.0) or t > 0.7
    assert math.isclose(magnitude, 0.1 * math.log(40.0) + 1.0)
    for bad in ({"kind": "cubic"}, {"kind": "linear"}, {"kind": "linear", "factor": 0.5}, {"kind": "yarn", "factor": 2.0},
                {"kind": "linear", "factor": 2.0, "original": 3}):
        with pytest.raises(ValueError):
            rotary_frequencies(64, scaling=bad)
    for dim in (0, 7, 514):
        with pytest.raises(ValueError):
            rotary_frequencies(dim)


def test_e4m3_codes_and_halves():
    codes = np.arange(127, dtype=np.uint8)
    values = fp8_e4m3_decode(codes).astype(np.float64)
    assert np.array_equal(draft.e4m3_bytes(values), codes)
    assert np.array_equal(draft.e4m3_bytes(-values), codes | 128)
    middle = (values[:-1] + values[1:]) / 2
    assert np.array_equal(draft.e4m3_bytes(middle), np.where(codes[:-1] % 2 == 0, codes[:-1], codes[1:]))
    rng = np.random.default_rng(0)
    latent = rng.standard_normal((3, 512)).astype(np.float32)
    latent[1, 128:256] = 0
    bytes_, scales = draft.stored_rows(latent)
    assert scales[1, 1] == 1.0 and not bytes_[1, 128:256].any()
    back = fp8_e4m3_decode(bytes_).reshape(3, 4, 128) * scales[:, :, None]
    assert np.all(np.abs(back.reshape(3, 512) - latent) <= np.abs(latent) * 2.0 ** -4 + scales.max() * 2.0 ** -10)


def test_attention_of_equal_logits_is_the_mean():
    rng = np.random.default_rng(1)
    rows = np.zeros((9, 656), np.uint8)
    rows[:, :512] = draft.e4m3_bytes(rng.uniform(-3, 3, (9, 512)).astype(np.float32))
    rows[:, 640:656] = np.asarray([0.5, 1, 2, 4], "<f4").view(np.uint8)
    sees = np.asarray([True, False] * 4 + [True])
    out, lse, _, _ = draft.tree_attention(np.zeros((2, 576)), rows, sees, 0.1)
    nope, _, scales = draft.row_parts(rows)
    assert np.allclose(out, (nope * np.repeat(scales, 128, 1))[sees].mean(0)) and np.allclose(lse, math.log(5))
    out, lse, _, _ = draft.tree_attention(np.zeros((2, 576)), rows, np.zeros(9, bool), 0.1)
    assert not out.any() and np.all(lse == -np.inf)


def test_ancestors():
    bits, depth = draft.ancestors([-1, 0, 0, 2, 1, -1, 5])
    assert bits == [1, 3, 5, 13, 19, 32, 96] and depth == [0, 1, 1, 2, 2, 0, 1]


def _distribution(first_tokens, weights, vocab):
    return np.bincount(first_tokens, weights=weights, minlength=vocab)


def test_a_verified_chain_is_distributed_as_the_target():
    rng = np.random.default_rng(2)
    vocab, grid = 5, 400
    p, q = rng.dirichlet(np.ones(vocab)), rng.dirichlet(np.ones(vocab))
    q[3] = 0.0
    q /= q.sum()
    u = (np.arange(grid) + 0.5) / grid
    got = np.zeros(vocab)
    for x in range(vocab):
        if q[x] == 0:
            continue
        accept = min(1.0, p[x] / q[x])
        for v in u:
            path, out = draft.verify(np.stack([p, p]), [0, x], None, np.stack([q, q]), [v, 0], 0.0)
            assert (len(path) == 2) == (v * q[x] < p[x])
            if len(path) == 2:
                got[x] += q[x] / grid
        refused = [draft.verify(np.stack([p, p]), [0, x], None, np.stack([q, q]), [1 - 1e-9, 0], v)[1][0] for v in u] \
            if accept < 1 else []
        for t in refused:
            got[t] += q[x] * (1 - accept) / grid
    assert np.allclose(got, p, atol=2.0 * vocab / grid)


def test_a_verified_tree_is_distributed_as_the_target():
    rng = np.random.default_rng(3)
    vocab, grid = 6, 100
    p = rng.dirichlet(np.ones(vocab), size=4)
    u = (np.arange(grid) + 0.5) / grid
    got = np.zeros(vocab)
    for v in u:
        for w in u:
            path, out = draft.verify(p, [0, 4, 2, 4], [-1, 0, 0, 0], None, [v, 0, 0, 0], w)
            assert 3 not in path  # the second child named 4 has nothing left
            got[out[0]] += 1 / grid ** 2
    assert np.allclose(got, p[0], atol=2.0 * vocab / grid)


def test_tables_model_undoes_and_refuses():
    t = draft.Tables(3, 4, 6, 300)
    stack = list(t.stack)
    cu, slots, positions, _, status = t.extend([130, 0, 100])
    assert (cu, status, t.lengths) == ([0, 130, 130, 230], 0, [130, 0, 100])
    assert slots[129] == 1 * 128 + 1 and slots[130] == 2 * 128 and slots[230] == -1 and positions[229] == 99
    t.truncate([0, 0, 0])
    assert t.stack == stack
    assert t.extend([299, 2, 1])[4] == 16 and t.lengths == [299, 0, 0]  # rows past the step's
    t.commit([1, 5, 5])
    assert t.lengths == [1, 0, 0] and len(t.stack) == 5
    assert t.extend([0, 200, 300])[4] == 16 and t.lengths == [1, 200, 0]
    t.commit([0, 200, 0])
    t.max_tokens = 2000
    cu, _, _, _, status = t.extend([1, 200, 500])
    assert status == 8 and t.lengths == [2, 400, 0]


def test_tables_model_makes_a_chain_visible():
    t = draft.Tables(2, 4, 8, 80)
    visible = t.extend([3, 70])[3]
    assert visible[:3] == [1, 3, 7] and visible[3:73] == [(1 << min(i, 64)) - 1 for i in range(1, 71)] and not any(visible[73:])
    assert visible[3:67] == draft.ancestors(range(-1, 63))[0]  # as a tree whose tokens each follow the one before


def test_a_target_that_falls_short_of_one_still_gives_a_token():
    bf16 = [0.10009765625, 0.8984375]  # bf16(0.1) and bf16(0.9)
    p = np.asarray([bf16 + [0.0]] * 4)
    for u, last in ((0.0, 0), (0.999, 1), (1 - 2.0 ** -24, 1)):
        path, out = draft.verify(p, [9, 0, 1, 0], [-1, 0, 0, 0], None, [u, 0, 0, 0], 0.5)
        assert out[0] == last and len(path) == (2 if u < 0.9 else 1)
    assert draft.verify(p, [9, 1, 0, 2], [-1, 0, 0, 0], None, [0.999, 0, 0, 0], 0.5) == ([0], [0])
    # A refused token one step of bf16 below its draft, the rest equal: max(p - q, 0) is 0.
    p, q = np.asarray([[0.5, 0.498046875]] * 2), np.asarray([[0.5, 0.5]] * 2)
    assert draft.verify(p, [0, 1], None, q, [0.9999, 0], 0.4) == ([0], [0])
    assert draft.verify(p, [0, 1], None, q, [0.9999, 0], 0.6) == ([0], [1])
    assert draft.verify(np.zeros((2, 2)), [0, 1], None, q, [0.9, 0], 0.6) == ([0], [-1])
    assert draft.verify(np.zeros((2, 2)), [0, 1], None, None, [0.9, 0], 0.6) == ([0], [-1])


def test_tokens_of_a_target_drafted_whole_are_distributed_as_it():
    """All of the target's tokens drafted as children, probabilities that sum to 1 - 2^-7: no token is missing, and
    none has more than its probability and the missing part."""
    p, grid = np.asarray([0.25, 0.5, 0.2421875]), 4096
    got = np.zeros(3)
    for u in (np.arange(grid) + 0.5) / grid:
        got[draft.verify(np.stack([p] * 4), [0, 2, 0, 1], [-1, 0, 0, 0], None, [u, 0, 0, 0], 0.0)[1][0]] += 1 / grid
    assert math.isclose(got.sum(), 1.0) and np.all(np.abs(got - p) <= (1 - p.sum()) + 1 / grid) and np.all(got >= p - 1 / grid)


def test_rows_of_the_smallest_and_largest_latents():
    latent = np.zeros((4, 512), np.float32)
    latent[0, ::128], latent[0, 5] = 3.1e-43, -1e-45  # over 448: 0 in 32 bits
    latent[1, ::128] = 3.2e-43                        # over 448: the least number there is
    latent[2, 3], latent[2, 4], latent[2, 128:256] = np.nan, 2.0, np.nan
    latent[3, 300], latent[3, 301] = -np.inf, 1.0
    bytes_, scales = draft.stored_rows(latent)
    assert np.all(scales[0] == 1) and not (bytes_[0] & 127).any()
    assert np.all(scales[1] == np.float32(1e-45)) and (bytes_[1] & 127).max() < 127
    assert scales[2].tolist() == [np.float32(2 / 448), 1, 1, 1] and np.all(bytes_[2, 128:256] & 127 == 127)
    assert bytes_[2, 3] & 127 == 127 and bytes_[2, 4] == 126
    assert np.isinf(scales[3, 2]) and bytes_[3, 300] & 127 == 127 and not (np.delete(bytes_[3], 300) & 127).any()
