"""GPU parity of the operators around a prompt chunk's layers (kvip_amd.ChunkAttention, NormRotary, TokenHistory,
LogitProcessor) against oracle/prompt.py, which works in 64 bits and derives the bounds that stand beside its
values. Whole numbers have to be equal. A rounding is off by at most half a step (bf16 2^-8, fp16 2^-11, fp32
2^-24, e4m3 2^-4 of the value)."""
import math

import numpy as np
import pytest

import kvip_amd
from kvip_amd.runtime import abi
from oracle import draft, prompt
from tests.test_gpu_draft import HALF_STEP, ROW, SCALE, device, dtype_of, host, random_parents, say
from tests.test_gpu_draft_rules import random_rows

pytestmark = pytest.mark.gpu
LOWEST = {"fp32": 2.0 ** -149, "bf16": 2.0 ** -133, "fp16": 2.0 ** -24}  # step between the smallest values


# --- attention -------------------------------------------------------------------------------


class Chunks:
    """Packed chunks over a shuffled cache: counts[b] new tokens, contexts[b] rows before them, `pad` rows behind the last
    token (more than 64 rows in all: not the business of tree attention)."""

    def __init__(self, torch, rng, counts, contexts, heads, *, stride=ROW, spare=2, pad=70):
        self.torch, self.counts, self.heads = torch, counts, heads
        self.lens = [c + n for c, n in zip(contexts, counts)]
        blocks = [-(-x // 128) for x in self.lens]
        self.pages = sum(blocks) + spare
        order, at = rng.permutation(self.pages), 0
        self.table = np.full((len(counts), max(max(blocks), 1)), -7, np.int32)  # entries past a request's pages are not read
        for b, n in enumerate(blocks):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.rows = np.full((self.pages * 128, stride), 0xFF, np.uint8)
        self.rows[:, :ROW] = random_rows(rng, self.pages * 128)
        used = np.zeros(len(self.rows), bool)
        for b in range(len(counts)):
            used[[self.slot(b, p) for p in range(self.lens[b])]] = True
        self.rows[~used] = 0xFF  # NaN features and scales in rows that nobody has
        self.tokens = sum(counts) + pad
        self.cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        gen = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
        self.query = torch.randn((self.tokens, heads, 576), generator=gen).to(torch.bfloat16)

    def slot(self, b, position):
        return self.table[b, position // 128] * 128 + position % 128

    def run(self, *, output="bf16", scale=SCALE, lse=True, steps=None, max_rows=None):
        torch = self.torch
        self.kv = torch.from_numpy(self.rows).cuda().view(self.pages, 128, -1)
        op = kvip_amd.ChunkAttention(torch, batch=len(self.counts), heads=self.heads, max_tokens=self.tokens,
                                     max_context=self.table.shape[1] * 128, max_rows=max_rows, device="cuda",
                                     output_dtype=dtype_of(torch, output), lse=lse)
        op.output.fill_(3.0)
        if lse:
            op.lse.fill_(3.0)
        return op.bind(self.query.cuda(), self.kv, device(torch, self.table, torch.int32), device(torch, self.lens, torch.int32),
                       device(torch, self.cu, torch.int32), scale,
                       steps=None if steps is None else device(torch, steps, torch.int32))

    def check(self, op, *, output="bf16", scale=SCALE, only=None, every=1):
        """Tokens i of a chunk with i % every == 0, the first and the last."""
        got = host(op())
        lse = None if op.lse is None else host(op.lse)
        q, worst = self.query.double().numpy(), 0.0
        for b, n in enumerate(self.counts):
            if only is not None and b not in only:
                continue
            key, value, odd = prompt.features(self.rows[[self.slot(b, p) for p in range(self.lens[b])]])
            assert not odd.any()
            for i in sorted({j for j in range(n) if j % every == 0} | {n - 1} if n else ()):
                row, sees = self.cu[b] + i, self.lens[b] - n + i + 1
                want, want_lse, bound, lse_bound = prompt.attention(q[row], key[:sees], value[:sees], scale)
                bound = bound + np.abs(want) * HALF_STEP[output]
                off = np.abs(got[row] - want)
                assert np.all(off <= bound), (b, i, float((off - bound).max()))
                worst = max(worst, float((off / np.maximum(bound, 1e-30)).max()))
                if lse is not None:
                    assert np.all(np.abs(lse[row] - want_lse) <= lse_bound), (b, i)
        say(f"  largest share of the bound {worst:.2f}")
        behind = self.cu[-1]
        assert np.all(got[behind:] == 3.0) and (lse is None or np.all(lse[behind:] == 3.0))


@pytest.mark.parametrize("heads,counts,contexts,every", [
    (1, [1], [0], 1), (16, [1], [0], 1), (16, [33], [0], 1), (16, [7, 0, 1], [32, 0, 31], 1), (5, [40, 3], [100, 129], 1),
    (128, [2, 1], [63, 500], 1), (20, [65], [255], 1), (3, [200], [0], 1), (16, [130], [900], 13), (8, [300, 1, 77], [0, 700, 2000], 17),
    (16, [1] * 40, list(range(0, 200, 5)), 1), (33, [64, 65, 127], [1, 127, 128], 9), (128, [70], [1000], 11), (7, [1000], [50], 97),
    (64, [400], [300], 41)])
def test_chunk_attention_matches(torch_gpu, heads, counts, contexts, every):
    say(f"case chunk heads={heads} counts={counts[:6]} contexts={contexts[:6]}")
    step = Chunks(torch_gpu, np.random.default_rng(heads + len(counts)), counts, contexts, heads)
    op = step.run()
    step.check(op, every=every)
    assert int(op.status.item()) == 0
    first = op.output.clone()
    assert torch_gpu.equal(op(), first)  # joined in one order


@pytest.mark.parametrize("heads,requests,most,longest", [(2, 300, 90, 700), (16, 60, 300, 1500), (128, 9, 40, 900), (1, 1024, 6, 300)])
def test_chunk_attention_of_many_requests(torch_gpu, heads, requests, most, longest):
    """More row tiles than workgroups, of requests with shared pages, and of some without tokens."""
    torch = torch_gpu
    say(f"case chunk many heads={heads} requests={requests}")
    rng = np.random.default_rng(requests)
    step = Chunks(torch, rng, [1], [127 + 128 * 39], heads, spare=0)
    step.counts = [int(rng.integers(1, most)) if rng.random() < 0.85 else 0 for _ in range(requests)]
    step.lens = [n + int(rng.integers(0, longest)) if rng.random() < 0.7 else n for n in step.counts]
    step.table = rng.integers(0, step.pages, (requests, -(-max(step.lens) // 128))).astype(np.int32)
    step.cu = np.concatenate([[0], np.cumsum(step.counts)]).astype(np.int32)
    step.tokens = int(step.cu[-1]) + 70
    step.query = torch.randn((step.tokens, heads, 576), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    op = step.run()
    step.check(op, every=41)
    assert int(op.status.item()) == 0


@pytest.mark.parametrize("heads,counts,contexts", [(16, [9], [30000]), (4, [3, 2], [40000, 100]), (128, [16], [9000]), (16, [100, 1], [20, 17000])])
def test_chunk_attention_cut_along_the_context(torch_gpu, heads, counts, contexts):
    say(f"case chunk cut heads={heads} counts={counts} contexts={contexts}")
    step = Chunks(torch_gpu, np.random.default_rng(heads), counts, contexts, heads)
    op = step.run()
    step.check(op, every=7)
    first = op.output.clone()
    assert torch_gpu.equal(op(), first)


@pytest.mark.parametrize("heads,counts,contexts", [(16, [1], [0]), (16, [30], [700]), (5, [40, 3, 0], [100, 129, 4]), (128, [2], [300]),
                                                   (16, [1] * 40, list(range(0, 200, 5)))])
def test_chunk_attention_of_few_rows(torch_gpu, heads, counts, contexts):
    """What tree attention carries out: its roundings, and its status bits."""
    torch = torch_gpu
    say(f"case chunk few heads={heads} counts={counts[:6]}")
    step = Chunks(torch, np.random.default_rng(heads), counts, contexts, heads, pad=2)
    op = step.run(max_rows=1)
    got, lse, q = host(op()), host(op.lse), step.query.double().numpy()
    for b, n in enumerate(counts):
        rows = step.rows[[step.slot(b, p) for p in range(step.lens[b])]]
        for i in range(n):
            sees = np.arange(len(rows)) <= step.lens[b] - n + i
            want, want_lse, bound, lse_bound = draft.tree_attention(q[step.cu[b] + i], rows, sees, SCALE)
            assert np.all(np.abs(got[step.cu[b] + i] - want) <= bound + np.abs(want) * 2.0 ** -8), (b, i)
            assert np.all(np.abs(lse[step.cu[b] + i] - want_lse) <= lse_bound), (b, i)
    assert np.all(got[step.cu[-1]:] == 3.0) and int(op.status.item()) == 0
    step.table[0, 0] = step.pages
    op = step.run(steps=[1] + [0] * (len(counts) - 1))
    op()
    assert int(op.status.item()) == abi.STATUS_BAD_BLOCK and not op.output[counts[0]:step.cu[-1]].any()


def test_chunk_attention_options(torch_gpu):
    """fp32 output without log-sum-exp, padded rows, other scales, and the functional form."""
    torch = torch_gpu
    say("case chunk options")
    step = Chunks(torch, np.random.default_rng(5), [90, 2], [60, 3000], 12, stride=720)
    op = step.run(output="fp32", scale=0.11, lse=False)
    step.check(op, output="fp32", scale=0.11, every=5)
    args = (step.query.cuda(), step.kv.view(step.pages, 128, 1, 720), device(torch, step.table, torch.int32),
            device(torch, step.lens, torch.int32), device(torch, step.cu, torch.int32))
    again = kvip_amd.chunk_attention(*args, scale=0.11, output_dtype=torch.float32)
    assert torch.equal(again[:92], op.output[:92])
    for scale in (-0.05, 0.0, 1e-30, 3e6):
        step.check(step.run(scale=scale), scale=scale, every=23)


def test_chunk_attention_of_nothing_but_zeros(torch_gpu):
    """Queries of zero weigh every row alike, under any scale."""
    torch = torch_gpu
    say("case chunk zero queries")
    step = Chunks(torch, np.random.default_rng(6), [50, 30], [200, 4000], 6)
    step.query[::2] = 0
    step.query[1::2] *= 1e-38  # logits that no scale brings to more than some units
    for scale in (3e38, -3e38, 1.0):
        step.check(step.run(scale=scale), scale=scale, every=7)


@pytest.mark.parametrize("heads,counts,contexts", [(4, [3], [200]), (16, [70, 9], [100, 700])])
def test_chunk_attention_takes_narrower_tables(torch_gpu, heads, counts, contexts):
    """An object for long contexts, bound to block tables of the step's."""
    torch = torch_gpu
    say(f"case chunk narrow table counts={counts}")
    step = Chunks(torch, np.random.default_rng(7), counts, contexts, heads, pad=0 if max(counts) < 64 else 70)
    first = step.run()()
    op = kvip_amd.ChunkAttention(torch, batch=len(counts), heads=heads, max_tokens=step.tokens, max_context=20000, max_rows=3000, device="cuda")
    args = (step.query.cuda(), step.kv, device(torch, step.table, torch.int32), device(torch, step.lens, torch.int32),
            device(torch, step.cu, torch.int32))
    got = op.bind(*args)()
    assert torch.equal(got[:sum(counts)], first[:sum(counts)])
    with pytest.raises(ValueError):
        op.bind(args[0], step.kv, torch.zeros((len(counts), 158), dtype=torch.int32, device="cuda"), *args[3:])


@pytest.mark.parametrize("heads,counts,contexts", [(16, [40], [500]), (16, [9, 60], [9000, 0])])
def test_chunk_attention_of_huge_logits(torch_gpu, heads, counts, contexts):
    """Logits of 10^7 and more: all weight is on the largest, and nothing overflows on the way."""
    torch = torch_gpu
    say(f"case chunk huge logits counts={counts}")
    step = Chunks(torch, np.random.default_rng(3), counts, contexts, heads)
    step.query = (step.query.float() * 2.0 ** 26).to(torch.bfloat16)
    op = step.run(output="fp32")
    got, lse, q, sure = host(op()), host(op.lse), step.query.double().numpy(), 0
    assert np.all(np.isfinite(got)) and np.all(np.isfinite(lse))
    for b, n in enumerate(counts):
        key, value, _ = prompt.features(step.rows[[step.slot(b, p) for p in range(step.lens[b])]])
        for i in range(0, n, 7):
            row, sees = step.cu[b] + i, step.lens[b] - n + i + 1
            logits = SCALE * (q[row] @ key[:sees].T)
            slip = SCALE * (np.abs(q[row]) @ np.abs(key[:sees]).T).max(1) * 584 * 2.0 ** -24
            top = logits.argmax(1)
            for h in range(heads):
                others = np.delete(logits[h], top[h])
                if len(others) and logits[h, top[h]] - others.max() < 2 * slip[h] + 100:
                    continue  # rounding may choose another
                sure += 1
                assert np.all(np.abs(got[row, h] - value[top[h]]) <= np.abs(value[top[h]]) * 2.0 ** -10), (b, i, h)
                assert abs(lse[row, h] - logits[h, top[h]]) <= slip[h] + abs(logits[h, top[h]]) * 2.0 ** -21
    assert sure > 50


def test_chunk_attention_equals_tree_attention_of_chains(torch_gpu):
    """Chains of up to 64 tokens are both operators' business; they round at other places, once or twice each."""
    torch = torch_gpu
    say("case chunk and tree")
    step = Chunks(torch, np.random.default_rng(8), [64, 5, 1], [300, 70, 900], 16)
    op = step.run(output="fp32")
    tree = kvip_amd.TreeAttention(torch, batch=3, heads=16, max_nodes=64, max_tokens=step.tokens, max_context=step.table.shape[1] * 128,
                                  device="cuda", output_dtype=torch.float32, lse=True)
    tree.bind(step.query.cuda(), step.kv, device(torch, step.table, torch.int32), device(torch, step.lens, torch.int32),
              device(torch, step.cu, torch.int32))
    a, b = op()[:70], tree()[:70]
    # Keys rounded to 2^-11 move a logit by at most 2^-11 scale sum |q k| (sum |q k| < 600 here, as 576 E|q k| is 367);
    # probabilities by twice that, values by 2^-11, this side's probabilities by 2^-11, the tree's by 2^-8.
    most = 2 ** -11 * (2 * 600 * SCALE + 3) + 2 ** -8
    key = [prompt.features(step.rows[[step.slot(i, p) for p in range(step.lens[i])]])[1] for i in range(3)]
    size = max(float(np.abs(k).max()) for k in key)
    assert float((a - b).abs().max()) <= most * size


@pytest.mark.parametrize("heads", [4, 16, 128])
def test_chunk_attention_hidden_rows_hold_anything(torch_gpu, heads):
    """NaN features, scales and rotary features, and infinite scales, in rows of the chunk that come after a token;
    tokens that see one of the first three are NaN."""
    torch = torch_gpu
    say(f"case chunk hidden heads={heads}")
    step = Chunks(torch, np.random.default_rng(heads), [50, 9, 40], [100, 700, 0], heads)
    clean = step.rows.copy()
    places = {0: (20, slice(640, 656), np.asarray([1, np.inf, 1, 2], "<f4").view(np.uint8)), 1: (4, slice(5, 9), [0x7F, 0xFF, 0x7F, 0x30]),
              2: (33, slice(512, 640), [0xFF] * 128)}
    for b, (i, where, what) in places.items():
        step.rows[step.slot(b, step.lens[b] - step.counts[b] + i), where] = what
    op = step.run()
    got, lse = host(op()), host(op.lse)
    step.rows = clean
    q = step.query.double().numpy()
    for b, n in enumerate(step.counts):
        key, value, _ = prompt.features(clean[[step.slot(b, p) for p in range(step.lens[b])]])
        for i in range(n):
            row = step.cu[b] + i
            if i >= places[b][0]:
                assert np.all(np.isnan(got[row])) and np.all(np.isnan(lse[row])), (b, i)
                continue
            sees = step.lens[b] - n + i + 1
            want, _, bound, _ = prompt.attention(q[row], key[:sees], value[:sees], SCALE)
            assert np.all(np.abs(got[row] - want) <= bound + np.abs(want) * 2.0 ** -8), (b, i)
    assert int(op.status.item()) == 0


@pytest.mark.parametrize("heads,counts,contexts", [(16, [70, 9], [100, 700]), (4, [40, 300], [0, 33])])
def test_chunk_attention_of_rows_of_other_sizes(torch_gpu, heads, counts, contexts):
    """Rows of a tile that are many orders of magnitude apart, those that a token sees and those that it does not, rows of
    zeros among them, and whole tiles that are larger or smaller than the others."""
    torch = torch_gpu
    say(f"case chunk sizes heads={heads}")
    rng = np.random.default_rng(heads)
    step = Chunks(torch, rng, counts, contexts, heads)
    scales = step.rows[:, 640:656].copy().view("<f4")
    for b, n in enumerate(counts):
        for p in range(step.lens[b]):
            at = step.slot(b, p)
            scales[at] *= 2.0 ** float(rng.integers(-30, 1) if p % 100 < 50 else -(p // 32 % 5) * 8)
            if p % 19 == 3:
                step.rows[at, :640] = 0
        for p in range(step.lens[b] - 5, step.lens[b]):
            scales[step.slot(b, p)] = 2.0 ** 60  # the last few: huge
    step.rows[:, 640:656] = scales.astype("<f4").view(np.uint8)
    op = step.run(output="fp32")
    got, q = host(op()), step.query.double().numpy()
    for b, n in enumerate(counts):
        key, value, odd = prompt.features(step.rows[[step.slot(b, p) for p in range(step.lens[b])]])
        assert not odd.any()
        for i in sorted({0, 1, 7, n // 2, n - 7, n - 6}):
            row, sees = step.cu[b] + i, step.lens[b] - n + i + 1
            want, _, bound, _ = prompt.attention(q[row], key[:sees], value[:sees], SCALE)
            # The probabilities' floor, under the largest exponent that a token has seen: 2^-36 of the largest value, as the
            # kernel's reference may be below the largest logit only, which raises them.
            floor = 2.0 ** -36 * sees * np.abs(value[:sees]).max()
            assert np.all(np.abs(got[row] - want) <= bound + np.abs(want) * 2.0 ** -24 + floor), (b, i)


def test_chunk_attention_bad_tables_and_lengths(torch_gpu):
    torch = torch_gpu
    say("case chunk bad tables")
    step = Chunks(torch, np.random.default_rng(9), [40, 2, 3], [470, 300, 200], 16)
    step.table[0, 1], step.table[0, 2] = step.pages, -1  # two of four pages are not there
    op = step.run()
    step.check(op, only=(1, 2))
    assert int(op.status.item()) == abi.STATUS_BAD_BLOCK
    q, got = step.query.double().numpy(), host(op.output)
    there = [p for p in range(510) if p // 128 not in (1, 2)]
    key, value, _ = prompt.features(step.rows[[step.slot(0, p) for p in there]], there)
    for i in (0, 39):
        n = sum(p <= 470 + i for p in there)
        want, _, bound, _ = prompt.attention(q[i], key[:n], value[:n], SCALE)
        assert np.all(np.abs(got[i] - want) <= bound + np.abs(want) * 2.0 ** -8)
    # Lengths past the table, below the chunk's tokens and below zero.
    step = Chunks(torch, np.random.default_rng(10), [2, 2, 3, 50], [500, 0, 100, 60], 16)
    step.lens[0], step.lens[1], step.lens[2] = 10 ** 6, 1, -5
    step.table[:] = np.maximum(step.table, 0)
    op = step.run()
    step.lens[0] = 0  # not looked at
    step.check(op, only=(3,), every=9)
    assert int(op.status.item()) == abi.STATUS_BAD_LENGTH
    assert not op.output[2].any() and bool((op.lse[2] == -math.inf).all())  # comes before the only row
    key, value, _ = prompt.features(step.rows[[step.slot(1, 0)]])
    assert np.all(np.abs(host(op.output[3]) - value) <= np.abs(value) * (2.0 ** -8 + 2.0 ** -10))
    assert not op.output[4:7].any()
    # cu_seqlens that fall and leave the rows.
    step = Chunks(torch, np.random.default_rng(12), [20, 30, 5], [100, 60, 7], 4)
    step.cu = np.asarray([0, 20, 10, 10 ** 6], np.int32)
    op = step.run()
    q, got = step.query.double().numpy(), host(op())
    key, value, _ = prompt.features(step.rows[[step.slot(0, p) for p in range(120)]])
    for i in (0, 9):
        want, _, bound, _ = prompt.attention(q[i], key[:101 + i], value[:101 + i], SCALE)
        assert np.all(np.abs(got[i] - want) <= bound + np.abs(want) * 2.0 ** -8)
    assert int(op.status.item()) == abi.STATUS_BAD_LENGTH


def test_chunk_attention_refused_requests(torch_gpu):
    """Requests that extend refused, and those that the workspace has no room for, get zeros."""
    torch = torch_gpu
    say("case chunk refused")
    step = Chunks(torch, np.random.default_rng(11), [40, 33, 7], [200, 90, 500], 16)
    op = step.run(steps=[40, 0, 7])
    step.check(op, only=(0, 2), every=6)
    assert not op.output[40:73].any() and bool((op.lse[40:73] == -math.inf).all()) and int(op.status.item()) == 0
    op = step.run(max_rows=512)  # 240 and 123 rows, then 507: 16 + 3 images' room, 8 + 4 + 16 needed
    step.check(op, only=(0, 1), every=6)
    assert not op.output[73:80].any() and bool((op.lse[73:80] == -math.inf).all())
    assert int(op.status.item()) == abi.STATUS_BAD_LENGTH


def test_chunk_attention_long_cache(torch_gpu):
    """Rows past the 4 GB of a cache, and images past the 4 GB of the workspace."""
    torch = torch_gpu
    say("case chunk long cache")
    step = Chunks(torch, np.random.default_rng(13), [5, 40], [2000, 700], 16)
    blocks, first = 60000, 60000 - step.pages  # 5.04 GB
    kv = torch.zeros((blocks, 128, ROW), dtype=torch.uint8, device="cuda")
    op = step.run()
    kv[first:] = step.kv
    op.bind(step.query.cuda(), kv, device(torch, step.table + first, torch.int32), device(torch, step.lens, torch.int32),
            device(torch, step.cu, torch.int32))
    step.check(op, every=9)
    del kv
    # A long request before the one that is looked at: 4.7 GB of images.
    long = 1 << 22
    table = torch.zeros((2, long // 128), dtype=torch.int32, device="cuda")
    table[1, :step.table.shape[1]] = device(torch, np.maximum(step.table[1], 0), torch.int32)
    op = kvip_amd.ChunkAttention(torch, batch=2, heads=16, max_tokens=101, max_context=long, max_rows=long + 1024, device="cuda")
    op.bind(step.query[4:105].cuda().contiguous(), step.kv, table, device(torch, [long, step.lens[1]], torch.int32),
            device(torch, [0, 1, 41], torch.int32))
    got, q = host(op()), step.query.double().numpy()[4:105]
    key, value, _ = prompt.features(step.rows[[step.slot(1, p) for p in range(step.lens[1])]])
    for i in (0, 17, 39):
        want, _, bound, _ = prompt.attention(q[1 + i], key[:701 + i], value[:701 + i], SCALE)
        assert np.all(np.abs(got[1 + i] - want) <= bound + np.abs(want) * 2.0 ** -8), i
    # The long one sees one page over and over: that page's attention.
    page = step.kv[0].cpu().numpy().reshape(128, -1)
    key, value, odd = prompt.features(page)
    if not odd.any():
        want, _, bound, _ = prompt.attention(q[0], key, value, SCALE)
        assert np.all(np.abs(got[0] - want) <= bound + np.abs(want) * (2.0 ** -8 + long * 2.0 ** -23))
    assert int(op.status.item()) == 0


def test_chunk_attention_refuses(torch_gpu):
    torch = torch_gpu
    op = kvip_amd.ChunkAttention(torch, batch=2, heads=4, max_tokens=6, max_context=256, device="cuda")
    good = dict(query=torch.zeros((6, 4, 576), dtype=torch.bfloat16, device="cuda"),
                kv_cache=torch.zeros((4, 128, 656), dtype=torch.uint8, device="cuda"),
                block_table=torch.zeros((2, 2), dtype=torch.int32, device="cuda"),
                seq_lens=torch.zeros(2, dtype=torch.int32, device="cuda"),
                cu_seqlens=torch.zeros(3, dtype=torch.int32, device="cuda"),
                steps=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        op()
    bad = dict(query=[good["query"].float(), good["query"][:5], good["query"].cpu(), good["query"].transpose(0, 1)],
               kv_cache=[good["kv_cache"].int(), good["kv_cache"][:, :64], good["kv_cache"][..., :640], good["kv_cache"].cpu()],
               block_table=[good["block_table"].long(), good["block_table"][:1], torch.zeros((2, 3), dtype=torch.int32, device="cuda"),
                            good["block_table"][:, :0]],
               seq_lens=[good["seq_lens"].long(), good["cu_seqlens"]], cu_seqlens=[good["seq_lens"], good["cu_seqlens"].long()],
               steps=[good["steps"].long(), good["cu_seqlens"]])
    for name, values in bad.items():
        for value in values:
            with pytest.raises(ValueError):
                op.bind(**{**good, name: value})
    for scale in (float("inf"), float("nan")):
        with pytest.raises(ValueError):
            op.bind(**good, scale=scale)
    assert not op.bind(**good)().any()  # a step without tokens


# --- norm and rotation -----------------------------------------------------------------------


def norm_case(torch, rng, dtype, tokens, heads, dim, skip):
    wide = device(torch, rng.standard_normal((tokens, heads, skip + dim)) * 1.5 + 0.3, dtype_of(torch, dtype))
    return wide[..., skip:]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("tokens,heads,keys,rotary,dim,norms", [
    (1, 1, 1, 64, 128, ("rms", "layer")), (5, 3, 2, 6, 7, ("layer", "rms")), (33, 16, 1, 64, 128, (None, "layer")),
    (7, 128, 4, 64, 64, ("rms", None)), (300, 2, 1, 32, 40, ("layer", "layer")), (2, 5, 1, 512, 512, ("rms", "rms")),
    (1500, 2, 1, 16, 24, ("layer", "rms")), (9, 4, 3, 64, 192, ("rms", "layer")), (40, 7, 1, 24, 256, ("layer", None)),
    (3, 2, 1, 2, 2, ("layer", "rms")), (4, 1, 1, 10, 511, ("rms", "layer"))])
def test_norm_rotary_matches(torch_gpu, dtype, half, tokens, heads, keys, rotary, dim, norms):
    torch = torch_gpu
    rng = np.random.default_rng(tokens * heads + dim)
    say(f"case norm {dtype} half={half} tokens={tokens} heads={heads} rotary={rotary} dim={dim} {norms}")
    t = dtype_of(torch, dtype)
    turn = kvip_amd.Rotary(torch, rotary_dim=rotary, layout="half" if half else "interleaved", device="cuda",
                           scaling={"kind": "yarn", "factor": 8.0, "original": 4096} if heads == 16 else None)
    op = kvip_amd.NormRotary(torch, rotary=turn, dim=dim, query_norm=norms[0], key_norm=norms[1], epsilon=1e-5)
    positions = rng.integers(0, 1 << 20, tokens)
    query, key = norm_case(torch, rng, dtype, tokens, heads, dim, 3), norm_case(torch, rng, dtype, tokens, keys, dim, 0)
    weights = {"query_weight": rng.standard_normal(dim) + 1, "query_bias": None, "key_weight": None if keys == 2 else
               rng.standard_normal(dim), "key_bias": rng.standard_normal(dim)}
    weights = {k: None if v is None else v.astype(np.float32) for k, v in weights.items()}
    x, k = host(query), host(key)
    out = torch.full((heads, tokens, dim + 1), 7.0, dtype=t, device="cuda")  # heads first, rows one apart
    y = out.transpose(0, 1)[..., :dim]
    op.bind(device(torch, positions, torch.int64), query, key, query_out=y,
            **{n: None if v is None else device(torch, v, torch.float32) for n, v in weights.items()})
    got, held = op()
    assert got is y and held is key
    frequencies = turn.frequencies.cpu().numpy()
    for have, from_, norm, what in ((y, x, norms[0], "query"), (key, k, norms[1], "key")):  # into another array, and in place
        want, bound = prompt.normed(from_, norm, weights[what + "_weight"], weights[what + "_bias"], 1e-5)
        want, bound = prompt.turned(want, bound, positions, frequencies, half, turn.magnitude)
        off = np.abs(host(have) - want)
        assert np.all(off <= bound + (np.abs(want) + bound) * HALF_STEP[dtype] + LOWEST[dtype]), (what, float(off.max()))
    assert torch.all(out[..., dim:] == 7.0) and np.array_equal(host(query), x) and int(op.status.item()) == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("half,rotary,tokens,heads", [(True, 64, 1, 64), (False, 64, 300, 32), (True, 128, 77, 5), (False, 20, 33, 3),
                                                      (True, 6, 130, 64)])
def test_index_heads_match(torch_gpu, dtype, half, rotary, tokens, heads):
    """fp8 features, scales and pages of the index cache, padded tokens, strided pages; the rest of the cache stays."""
    torch = torch_gpu
    rng = np.random.default_rng(tokens + heads)
    say(f"case index heads {dtype} half={half} rotary={rotary} tokens={tokens} heads={heads}")
    turn = kvip_amd.Rotary(torch, rotary_dim=rotary, layout="half" if half else "interleaved", device="cuda")
    op = kvip_amd.NormRotary(torch, rotary=turn, dim=128, key_norm="layer")
    query, key = norm_case(torch, rng, dtype, tokens, heads, 128, 0), norm_case(torch, rng, dtype, tokens, 1, 128, 5)[:, 0]
    query[tokens // 2, 0] = 0.0
    weight, bias = (rng.standard_normal(128).astype(np.float32) for _ in range(2))
    blocks = -(-tokens // 128) + 2
    pages = torch.full((blocks, 2, 128, 128), 5, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, 1]
    scales = torch.full((blocks, 130), 9.0, device="cuda")[:, :128]
    slots = rng.permutation(blocks * 128)[:tokens]
    slots[::7] = -1
    positions = rng.integers(0, 100000, tokens)
    out = torch.empty((tokens, heads, 128), dtype=torch.float8_e4m3fn, device="cuda")
    scale = torch.empty((tokens, heads), device="cuda")
    op.bind(device(torch, positions, torch.int64), query, key, key_weight=device(torch, weight, torch.float32),
            key_bias=device(torch, bias, torch.float32), query_out=out, query_scale=scale, slots=device(torch, slots, torch.int64),
            key_cache=pages, key_scales=scales)
    assert op() == (out, pages)
    frequencies = turn.frequencies.cpu().numpy()

    def check(values, factor, want, bound, what):
        # The largest magnitude is off by its bound, the quotient by half a step; a feature by its own bound, its quotient by
        # half a step and the scale's error, then by half a step of its code.
        _, exact = prompt.codes(want)
        zero = np.abs(want).max(-1) == 0
        slack = np.where(zero, 0, bound.max(-1) / 448 + exact * 2.0 ** -23)
        assert np.all(np.abs(factor - exact) <= slack), what
        x = np.abs(want) + bound
        off = np.abs(values * factor[..., None] - want)
        limit = bound + x * (slack / exact + 2.0 ** -23)[..., None]
        limit = limit + np.maximum((x + limit) * 2.0 ** -4, factor[..., None] * 2.0 ** -10) * (1 + 2.0 ** -20)
        assert np.all(off <= limit), (what, float((off - limit).max()))

    zero = np.zeros((tokens, heads, 128))
    want, bound = prompt.turned(host(query), zero, positions, frequencies, half, turn.magnitude)
    check(host(out.float()), host(scale), want, bound, "query")
    assert not out[tokens // 2, 0].float().any() and float(scale[tokens // 2, 0]) == 1.0
    want, bound = prompt.normed(host(key), "layer", weight, bias)
    want, bound = prompt.turned(want, bound, positions, frequencies, half, turn.magnitude)
    held, kept = pages.float().reshape(-1, 128).cpu().numpy(), slots >= 0
    per_key = scales.reshape(-1).cpu().numpy()
    check(held[slots[kept]].astype(np.float64), per_key[slots[kept]].astype(np.float64), want[kept], bound[kept], "key")
    rest = np.setdiff1d(np.arange(blocks * 128), slots[kept])
    assert np.all(pages.view(torch.uint8).reshape(-1, 128).cpu().numpy()[rest] == 5) and np.all(per_key[rest] == 9.0)
    assert int(op.status.item()) == 0


def test_index_heads_edges(torch_gpu):
    """NaN and infinite features, the smallest magnitudes, a slot past the cache."""
    torch = torch_gpu
    say("case index edges")
    turn = kvip_amd.Rotary(torch, rotary_dim=64, device="cuda")
    op = kvip_amd.NormRotary(torch, rotary=turn, dim=128)
    x = torch.zeros((5, 1, 128), device="cuda")
    x[0, 0, 100], x[0, 0, 101] = math.nan, 2.0
    x[1, 0, 100], x[1, 0, 101] = math.inf, 2.0
    x[2, 0, 100] = 1e-44
    x[3, 0, 100], x[3, 0, 101] = 3e38, -1e38
    out, scale = torch.zeros((5, 1, 128), dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros((5, 1), device="cuda")
    pages, scales = torch.zeros((2, 128, 128), dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros((2, 128), device="cuda")
    slots = torch.tensor([0, 1, 255, 256, -5], device="cuda")
    op.bind(torch.zeros(5, dtype=torch.int64, device="cuda"), x, x[:, 0].clone(), query_out=out, query_scale=scale, slots=slots,
            key_cache=pages, key_scales=scales)()
    y = out.float()[:, 0]
    assert bool(y[0, 100].isnan()) and float(y[0, 101]) == 448.0 and abs(float(scale[0]) * 448 - 2) < 1e-6
    assert bool(y[1, 100].isnan()) and float(y[1, 101]) == 0.0 and float(scale[1]) == math.inf
    assert float(scale[2]) == 1.0 and not y[2].any()
    assert float(y[3, 100]) == 448.0 and float(y[3, 101]) in (-144.0, -160.0)
    assert int(op.status.item()) == abi.STATUS_BAD_TOKEN and not pages.float()[1, :127].any() and float(scales[1, 127]) == 1.0


def test_norm_rotary_of_more_heads_than_a_launch(torch_gpu):
    torch = torch_gpu
    say("case norm of 2^20 + 3 tokens x 32 heads")
    n = (1 << 20) + 3
    turn = kvip_amd.Rotary(torch, rotary_dim=2, device="cuda")
    x = torch.randn((1, 1, 8), device="cuda").expand(n, 32, 8)
    y = torch.empty((n, 32, 8), device="cuda")
    op = kvip_amd.NormRotary(torch, rotary=kvip_amd.Rotary(torch, rotary_dim=8, device="cuda"), dim=8, query_norm="rms")
    op.bind(torch.arange(n, device="cuda") % 1000, x, query_out=y)()
    assert torch.equal(y[1000:], y[:n - 1000]) and torch.equal(y[:, :1].expand(n, 32, 8), y) and not torch.equal(y[0], y[1])
    z = torch.empty((n, 3), device="cuda")
    op = kvip_amd.NormRotary(torch, rotary=turn, dim=3, query_norm="layer")
    op.bind(torch.arange(n, device="cuda") % 1000, x[:, 0, :3], query_out=z)()
    assert torch.equal(z[1000:], z[:n - 1000]) and not torch.equal(z[0], z[1])


def test_norm_rotary_refuses(torch_gpu):
    torch = torch_gpu
    turn = kvip_amd.Rotary(torch, rotary_dim=8, device="cuda")
    op = kvip_amd.NormRotary(torch, rotary=turn, dim=16, query_norm="rms")
    positions = torch.zeros(4, dtype=torch.int64, device="cuda")
    x = torch.zeros((4, 2, 16), dtype=torch.bfloat16, device="cuda")
    w = torch.ones(16, device="cuda")
    with pytest.raises(ValueError):
        op()
    for query, kw in ((x[:3], {}), (x[..., :8], {}), (x.double(), {}), (x.cpu(), {}), (x.transpose(1, 2), {}),
                      (x, dict(key=x.float())), (x, dict(key_out=x)), (x, dict(key_weight=w)), (x, dict(query_out=x.float())),
                      (x, dict(query_out=x[:, :1].expand(4, 2, 16))), (x[:, :1].expand(4, 2, 16), {}), (x, dict(query_weight=w[:8])),
                      (x, dict(query_weight=w.bfloat16())), (x, dict(query_bias=w.cpu())), (x, dict(slots=positions)),
                      (x, dict(query_scale=torch.zeros((4, 2), device="cuda")))):
        with pytest.raises(ValueError):
            op.bind(positions, query, **kw)
    for bad in (positions.int(), positions.cpu(), positions.view(2, 2)):
        with pytest.raises(ValueError):
            op.bind(bad, x)
    op = kvip_amd.NormRotary(torch, rotary=turn, dim=128)
    q = torch.zeros((4, 2, 128), dtype=torch.bfloat16, device="cuda")
    good = dict(key=q[:, 0], query_out=torch.zeros((4, 2, 128), dtype=torch.float8_e4m3fn, device="cuda"),
                query_scale=torch.zeros((4, 2), device="cuda"), slots=positions,
                key_cache=torch.zeros((2, 128, 128), dtype=torch.float8_e4m3fn, device="cuda"),
                key_scales=torch.zeros((2, 128), device="cuda"))
    bad = dict(key=[q], query_out=[None, q, good["query_out"][:, :1]], query_scale=[None, good["query_scale"][:3], good["query_scale"].double()],
               slots=[None, positions.int(), positions[:3]], key_cache=[None, good["key_cache"][:, :64], good["key_cache"].float()],
               key_scales=[None, good["key_scales"][:1], good["key_scales"].double()], key_out=[q[:, 0]])
    for name, values in bad.items():
        for value in values:
            with pytest.raises(ValueError):
                op.bind(positions, q, **{**good, name: value})
    none = {k: v[:0] if k in ("key", "query_out", "query_scale", "slots") else v for k, v in good.items()}
    op.bind(positions[:0], q[:0], **none)()  # no tokens


# --- logits ----------------------------------------------------------------------------------


def load_histories(torch, rng, op, model, lengths):
    vocab, batch = model.vocab, len(lengths)
    order = rng.permutation(batch)
    tokens = [rng.integers(0, max(1, vocab // 3), n) for n in lengths]
    prompts = [n // 2 for n in lengths]
    cu = np.concatenate([[0], np.cumsum(lengths)])
    op.load(device(torch, order, torch.int32), device(torch, np.concatenate(tokens), torch.int64), device(torch, cu, torch.int32),
            device(torch, prompts, torch.int32))
    for i, b in enumerate(order):
        model.load(b, tokens[i], prompts[i])


def same_history(op, model):
    counts, seen = model.arrays()
    assert np.array_equal(op.counts.cpu().numpy(), counts) and np.array_equal(op.seen.cpu().numpy(), seen)


@pytest.mark.parametrize("vocab,lengths", [(1, [3]), (31, [0, 5]), (33, [100, 1, 7]), (16384, [5000]), (16385, [20, 3000]),
                                           (50001, [0, 0, 900, 40000]), (1 << 20, [70, 9000])])
def test_histories_follow_the_model(torch_gpu, vocab, lengths):
    torch = torch_gpu
    say(f"case history vocab={vocab} lengths={lengths}")
    rng, batch = np.random.default_rng(vocab), len(lengths)
    op, model = kvip_amd.TokenHistory(torch, batch=batch, vocab=vocab, device="cuda"), prompt.History(batch, vocab)
    load_histories(torch, rng, op, model, lengths)
    same_history(op, model)
    for places in (1, 5, 64):
        tokens, kept = rng.integers(0, vocab, (batch, places)), rng.integers(0, places + 1, batch)
        tokens[:, places // 2:] = tokens[:, :1]  # one token several times
        op.append(device(torch, tokens, torch.int64), device(torch, kept, torch.int32))
        for b in range(batch):
            model.append(b, tokens[b, :kept[b]])
        same_history(op, model)
    # One request starts over, the others stay; tokens and requests that are not there.
    op.load(device(torch, [-1, 0], torch.int32), device(torch, [0, vocab, -1, 0, 0], torch.int64),
            device(torch, [0, 1, 5], torch.int32), device(torch, [0, 3], torch.int32))
    model.load(0, [vocab, -1, 0, 0], 3)
    same_history(op, model)
    assert int(op.status.item()) == abi.STATUS_BAD_TOKEN
    op.status.zero_()
    op.load(device(torch, [batch, 0], torch.int32), device(torch, [0, 0], torch.int64), device(torch, [0, 1, 9], torch.int32),
            device(torch, [0, 0], torch.int32))
    model.load(0, [0], 0)
    same_history(op, model)
    assert int(op.status.item()) == abi.STATUS_BAD_LENGTH
    op.load(device(torch, [0], torch.int32), torch.zeros(0, dtype=torch.int64, device="cuda"), device(torch, [0, 0], torch.int32),
            device(torch, [0], torch.int32))
    model.load(0, [], 0)
    same_history(op, model)
    op.status.zero_()
    op.append(device(torch, np.full((batch, 2), vocab), torch.int64), device(torch, np.full(batch, 3), torch.int32))
    same_history(op, model)
    assert int(op.status.item()) == abi.STATUS_BAD_TOKEN | abi.STATUS_BAD_LENGTH


class Sampling:
    """A packed step's rows with everything that may bear on them."""

    def __init__(self, torch, rng, counts, vocab, dtype, *, biases=0, masked=False, history=True, trees=True, output="fp32", pad=2,
                 width=0):
        batch = len(counts)
        self.torch, self.counts, self.vocab, self.output = torch, counts, vocab, output
        self.cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.rows = int(self.cu[-1]) + pad
        wide = torch.zeros((self.rows, vocab + width), dtype=dtype_of(torch, dtype), device="cuda")
        self.logits = wide[:, :vocab]
        self.logits.copy_(torch.from_numpy(rng.standard_normal((self.rows, vocab)) * 4))
        self.tokens = rng.integers(0, vocab, self.rows)
        parents = random_parents(rng, counts, self.rows) if trees else np.zeros(self.rows, np.int32)
        self.visible = np.zeros(self.rows, np.uint64)
        for b, n in enumerate(counts):
            at = slice(self.cu[b], self.cu[b] + n)
            self.visible[at] = np.asarray(draft.ancestors(parents[at].tolist())[0], np.uint64)[:n] if n else []
            if n > 4:
                self.tokens[self.cu[b] + 1:self.cu[b] + 4] = self.tokens[self.cu[b]]  # one token several times on a way

        def per_request(low, high):
            return rng.uniform(low, high, batch).astype(np.float32)

        self.numbers = {"temperature": per_request(0.3, 2.0), "repetition": per_request(0.7, 1.6), "presence": per_request(-0.5, 1.0),
                        "frequency": per_request(-0.1, 0.4)}
        self.numbers["temperature"][1::4] = 0.0
        self.names = self.values = self.allowed = None
        if biases:
            self.names, self.values = rng.integers(-1, vocab, (batch, biases)), rng.uniform(-5, 5, (batch, biases)).astype(np.float32)
            self.names[:, biases // 2] = self.names[:, 0]  # named twice
            self.names[:, -1] = self.tokens[np.minimum(self.cu[:-1] + 1, self.rows - 1)]  # a drafted one
        if masked:
            self.allowed = rng.integers(-2 ** 31, 2 ** 31, (self.rows, -(-vocab // 32))) & rng.integers(-2 ** 31, 2 ** 31, (self.rows, -(-vocab // 32)))
        self.model = prompt.History(batch, vocab) if history else None
        self.history = kvip_amd.TokenHistory(torch, batch=batch, vocab=vocab, device="cuda") if history else None
        if history:
            load_histories(torch, rng, self.history, self.model, rng.integers(0, 3 * vocab if vocab < 500 else 900, batch).tolist())

    def op(self, **changed):
        torch, n = self.torch, self.numbers
        op = kvip_amd.LogitProcessor(torch, batch=len(self.counts), max_tokens=self.rows, vocab=self.vocab, device="cuda",
                                     output_dtype=dtype_of(torch, self.output))
        op.probs.fill_(3.0)
        kw = {k: device(torch, v, torch.float32) for k, v in n.items()}
        kw.update(history=self.history, tokens=device(torch, self.tokens, torch.int64),
                  visible=device(torch, self.visible.view(np.int64), torch.int64))
        if self.names is not None:
            kw.update(bias_tokens=device(torch, self.names, torch.int32), bias_values=device(torch, self.values, torch.float32))
        if self.allowed is not None:
            kw.update(allowed=device(torch, self.allowed, torch.int32))
        return op.bind(self.logits, device(torch, self.cu, torch.int32), **{**kw, **changed})

    def row(self, b, i, x):
        """(probabilities, bound, adjusted logits, bound, odd) of row i of request b with logits x."""
        row = self.cu[b] + i
        way = [int(self.tokens[self.cu[b] + j]) for j in range(1, self.counts[b]) if int(self.visible[row]) >> j & 1]
        allowed = None
        if self.allowed is not None:
            words = self.allowed[row].astype(np.int64)[:, None] >> np.arange(32)
            allowed = (words & 1).astype(bool).reshape(-1)[:self.vocab]
        n = {k: float(v[b]) for k, v in self.numbers.items()}
        z, bound, odd = prompt.logits(
            x, wrote=self.model.wrote[b] if self.model else None, has=self.model.has[b] if self.model else None, way=way,
            repetition=n["repetition"], presence=n["presence"], frequency=n["frequency"],
            biases=[] if self.names is None else list(zip(self.names[b].tolist(), self.values[b].tolist())), allowed=allowed)
        return (*prompt.probabilities(z, bound, n["temperature"]), z, bound, odd)

    def check(self, got, rows=None):
        x, worst = host(self.logits), 0.0
        got = host(got)
        for b, n in enumerate(self.counts):
            for i in range(n):
                row = self.cu[b] + i
                p, bound, z, slip, _ = self.row(b, i, x[row])
                if not self.numbers["temperature"][b] > 0:
                    at = int(np.argmax(got[row]))  # of those that rounding cannot tell from the largest, exactly one
                    assert got[row, at] == 1.0 and np.count_nonzero(got[row]) == 1
                    assert z[at] + slip[at] >= np.max(z - slip), (b, i)
                    if slip.max() == 0:
                        assert at == int(np.argmax(z)), (b, i)
                    continue
                limit = bound + p * HALF_STEP[self.output] + LOWEST[self.output]
                off = np.abs(got[row] - p)
                assert np.all(off <= limit), (b, i, float((off - limit).max()))
                worst = max(worst, float((off / np.maximum(limit, 1e-38)).max()))
        say(f"  largest share of the bound {worst:.2f}")
        assert np.all(got[self.cu[-1]:] == 3.0)


@pytest.mark.parametrize("dtype,output", [("fp32", "fp32"), ("bf16", "fp32"), ("fp16", "bf16"), ("bf16", "fp16")])
@pytest.mark.parametrize("counts,vocab,biases,masked", [
    ([1], 1, 0, False), ([1], 9, 1, False), ([3, 0, 5], 33, 4, True), ([64], 700, 0, False), ([7, 1, 1, 20], 4097, 40, True),
    ([1, 2], 32000, 300, True), ([1], 131073, 20, False), ([5] * 9, 5003, 0, True)])
def test_probabilities_match(torch_gpu, dtype, output, counts, vocab, biases, masked):
    say(f"case logits {dtype} to {output} counts={counts} vocab={vocab} biases={biases} masked={masked}")
    s = Sampling(torch_gpu, np.random.default_rng(vocab + len(counts)), counts, vocab, dtype, biases=biases, masked=masked,
                 output=output, width=3)
    if masked:
        s.allowed[:, 0] |= 1  # no row without any token
    op = s.op()
    got = op()
    s.check(got)
    assert int(op.status.item()) == 0
    first = got.clone()
    assert torch_gpu.equal(op(), first)


@pytest.mark.parametrize("rows,vocab", [(300, 9000), (1100, 131072 // 16), (40, 40000), (1030, 200000 // 8), (1200, 140001)])
def test_probabilities_of_many_rows(torch_gpu, rows, vocab):
    """Rows that one workgroup takes whole, and those that several take; rows of more tokens than a workgroup takes."""
    torch = torch_gpu
    say(f"case logits rows={rows} vocab={vocab}")
    counts = [1] * 20 + [20] * ((rows - 20) // 20)
    s = Sampling(torch, np.random.default_rng(rows), counts, vocab, "bf16", biases=9)
    op = s.op()
    got = op()
    x = s.logits.double()
    for b in (0, 1, 19, 20, len(counts) - 1):
        for i in {0, counts[b] - 1}:
            row = s.cu[b] + i
            p, bound, z, slip, _ = s.row(b, i, x[row].cpu().numpy())
            have = host(got[row])
            if s.numbers["temperature"][b] > 0:
                assert np.all(np.abs(have - p) <= bound + LOWEST["fp32"] + p * 2.0 ** -24), (b, i)
            else:
                at = int(np.argmax(have))
                assert have[at] == 1.0 and np.count_nonzero(have) == 1 and z[at] + slip[at] >= np.max(z - slip)
    sums = got[:s.cu[-1]].double().sum(1)
    assert float((sums - 1).abs().max()) <= 2.0 ** -13
    assert bool((got[s.cu[-1]:] == 3.0).all()) and int(op.status.item()) == 0


def test_logits_alone(torch_gpu):
    """Nothing but logits: a softmax; nothing but a temperature of 0: the first of the largest."""
    torch = torch_gpu
    say("case logits alone")
    s = Sampling(torch, np.random.default_rng(1), [3, 2], 500, "bf16", history=False, trees=False)
    s.logits[0, 100:103] = 40.0
    none = dict(temperature=None, repetition=None, presence=None, frequency=None, tokens=None, visible=None)
    s.numbers = {"temperature": np.ones(2), "repetition": np.ones(2), "presence": np.zeros(2), "frequency": np.zeros(2)}
    s.visible[:] = 0
    s.check(s.op(**none)())
    zero = torch.tensor([0.0, -1.0], device="cuda")
    got = s.op(**{**none, "temperature": zero})()
    s.numbers["temperature"] = np.zeros(2)
    s.check(got)
    assert float(got[0, 100]) == 1.0
    # Temperatures that are no ordinary numbers.
    got = s.op(**{**none, "temperature": torch.tensor([1e-42, math.inf], device="cuda")})()
    assert float((got[0, 100:103] - 1 / 3).abs().max()) < 1e-6 and float((got[3:5] * 500 - 1).abs().max()) < 1e-5
    got = s.op(**{**none, "temperature": torch.tensor([math.nan, 1.0], device="cuda")})()
    assert float(got[0, 100]) == 1.0


@pytest.mark.parametrize("vocab", [40, 9001])
def test_masked_and_odd_logits(torch_gpu, vocab):
    """Rows that a mask leaves nothing, masks of the type's lowest value, infinities, and NaN in masked places."""
    torch = torch_gpu
    say(f"case odd logits vocab={vocab}")
    s = Sampling(torch, np.random.default_rng(vocab), [9], vocab, "fp32", masked=True, biases=2)
    s.numbers["temperature"][:], s.numbers["repetition"][:] = 0.7, 1.0  # times 1.5 the lowest value would pass the range
    s.names[0], s.values[0] = [3, 4], [-math.inf, 1.0]
    s.allowed[:] = -1
    s.allowed[0] = 0                                    # nothing allowed
    s.allowed[1] = 0
    s.allowed[1, 0] = 1 << 3 | 1 << 4                   # a banned token and another
    s.logits[2, 5:] = torch.finfo(torch.float32).min    # masked by the lowest value
    s.logits[3] = torch.finfo(torch.float32).min        # all of them
    s.logits[4] = -math.inf                             # all of them
    s.logits[5, 7], s.logits[5, 9] = math.inf, math.inf
    s.logits[6, 11] = math.nan
    s.allowed[6, 0] &= ~(1 << 11)                       # a NaN that is masked
    s.logits[7, 12] = math.nan                          # one that is not
    s.logits[8, 13] = -math.inf
    op = s.op()
    got = host(op())
    for i in range(9):
        p, bound, _, _, odd = s.row(0, i, host(s.logits)[i])
        assert odd == (i == 7)
        assert np.all(np.abs(got[i] - p) <= bound + LOWEST["fp32"] + p * 2.0 ** -24), i
    assert not got[0].any() and got[1, 4] == 1.0 and not got[4].any() and abs(got[5, 7] - 0.5) < 1e-6
    assert int(op.status.item()) == abi.STATUS_BAD_PROBS
    s.logits[4], s.logits[7] = 0.0, 0.0
    s.allowed[0] = -1
    op = s.op()
    op()
    assert int(op.status.item()) == 0


@pytest.mark.parametrize("counts,vocab,biases", [([1], 9001, 30), ([6, 1], 32000, 64), ([5], 5000, 4096), ([3, 3], 140001, 4096), ([20], 64, 20)])
def test_lists_of_tokens_named_once_or_more(torch_gpu, counts, vocab, biases):
    """Biases of tokens that nothing else names, of drafted tokens, and of a token named by every third entry."""
    torch = torch_gpu
    say(f"case lists counts={counts} vocab={vocab} biases={biases}")
    rng = np.random.default_rng(vocab + biases)
    s = Sampling(torch, rng, counts, vocab, "fp32", biases=biases, masked=True)
    s.numbers["temperature"][:] = 0.8
    s.allowed[:, 0] |= 1
    drafted = set(s.tokens.tolist())
    for _ in range(2):
        for b in range(len(counts)):
            s.names[b] = rng.permutation([v for v in range(vocab) if v not in drafted or vocab < 100])[:biases]
        op = s.op()
        s.check(op())
        assert int(op.status.item()) == 0
        drafted = set()
    s.names[:, 1:biases // 2:7] = s.tokens[s.cu[:-1], None]
    op = s.op()
    s.check(op())
    s.names[:, ::3] = s.names[:, :1]
    op = s.op()
    s.check(op())
    assert int(op.status.item()) == 0


def test_logits_report(torch_gpu):
    torch = torch_gpu
    say("case logits report")
    s = Sampling(torch, np.random.default_rng(2), [5, 4], 100, "fp32", biases=3)
    s.names[0, 1] = 100
    op = s.op()
    s.check(op())  # the model leaves it out as well
    assert int(op.status.item()) == abi.STATUS_BAD_TOKEN
    s.names[0, 1] = 99
    s.tokens[1], s.tokens[2] = -1, 100
    op = s.op()
    s.check(op())
    assert int(op.status.item()) == abi.STATUS_BAD_TOKEN
    s.tokens[1:3] = 5
    op = s.op()
    op.bind(s.logits, device(torch, [0, 5, 1000], torch.int32))
    got = op()
    assert int(op.status.item()) == abi.STATUS_BAD_LENGTH
    assert float((got.double().sum(1) - 1).abs().max()) < 1e-5  # rows 9 and 10 are the second request's now
    op = s.op()
    op.bind(s.logits, device(torch, [3, 2, 8], torch.int32))
    got = op()
    assert int(op.status.item()) == abi.STATUS_BAD_LENGTH
    assert bool((got[:2] == 3.0).all()) and bool((got[8:] == 3.0).all()) and float((got[2:8].double().sum(1) - 1).abs().max()) < 1e-5


def test_logits_refuse(torch_gpu):
    torch = torch_gpu
    s = Sampling(torch, np.random.default_rng(3), [3, 2], 100, "fp32", biases=3, masked=True)
    op = s.op()
    with pytest.raises(ValueError):
        kvip_amd.LogitProcessor(torch, batch=2, max_tokens=7, vocab=100, device="cuda")()
    good = torch.zeros(2, device="cuda")
    bad = dict(temperature=[good[:1], good.double(), good.cpu()], repetition=[good.int()], presence=[good[:1]], frequency=[good.half()],
               tokens=[None, torch.zeros(7, dtype=torch.int32, device="cuda")], visible=[None, torch.zeros(6, dtype=torch.int64, device="cuda")],
               history=[kvip_amd.TokenHistory(torch, batch=3, vocab=100, device="cuda"), kvip_amd.TokenHistory(torch, batch=2, vocab=99, device="cuda")],
               bias_tokens=[None, torch.zeros((2, 4), dtype=torch.int32, device="cuda"), torch.zeros((2, 3), dtype=torch.int64, device="cuda"),
                            torch.zeros((2, 4097), dtype=torch.int32, device="cuda")],
               bias_values=[None, torch.zeros((2, 4), device="cuda")],
               allowed=[torch.zeros((7, 3), dtype=torch.int32, device="cuda"), torch.zeros((7, 4), dtype=torch.int64, device="cuda")])
    for name, values in bad.items():
        for value in values:
            with pytest.raises(ValueError):
                s.op(**{name: value})
    cu = device(torch, s.cu, torch.int32)
    for logits in (s.logits[:6], s.logits[:, :99], s.logits.double(), s.logits.cpu(), s.logits.t(), op.probs,
                   torch.zeros((100, 7), device="cuda").t()):
        with pytest.raises(ValueError):
            op.bind(logits, cu)
    with pytest.raises(ValueError):
        op.bind(s.logits, cu.long())
    h = s.history
    for args in ((cu[:2].long(), cu.long(), cu, cu[:2]), (cu[:2], cu, cu, cu[:2]), (cu[:2], cu.long(), cu[:2], cu[:2]),
                 (cu[:2], cu.long(), cu, cu), (cu[:0], cu.long(), cu[:1], cu[:0])):
        with pytest.raises(ValueError):
            h.load(*args)
    tokens = torch.zeros((2, 4), dtype=torch.int64, device="cuda")
    for args in ((tokens.int(), cu[:2]), (tokens, cu), (tokens[:1], cu[:1]), (torch.zeros((2, 65), dtype=torch.int64, device="cuda"), cu[:2])):
        with pytest.raises(ValueError):
            h.append(*args)


# --- all of them together --------------------------------------------------------------------


class Prompts:
    """Chunks of three requests through one layer and the sampler, then steps of drafted chains, over one cache."""

    HEADS, INDEX, VOCAB, ROWS, NODES = 12, 32, 700, 330, 6

    def __init__(self, torch, seed):
        self.torch = torch
        rng, z = np.random.default_rng(seed), lambda *shape: torch.zeros(shape, device="cuda")
        rows, bf = self.ROWS, torch.bfloat16
        self.kv = torch.zeros((12, 128, ROW), dtype=torch.uint8, device="cuda")
        self.index_keys = torch.zeros((12, 128, 128), dtype=torch.float8_e4m3fn, device="cuda")
        self.index_scales = z(12, 128)
        self.tables = kvip_amd.PageTables(torch, batch=3, max_context=768, num_blocks=12, max_tokens=rows, device="cuda",
                                          caches=[self.kv, self.index_keys, self.index_scales])
        self.latent, self.rope, self.query = z(rows, 512).to(bf), z(rows, 64).to(bf), z(rows, self.HEADS, 576).to(bf)
        self.index_q, self.index_k = z(rows, self.INDEX, 128).to(bf), z(rows, 1, 128).to(bf)
        self.index_codes = torch.zeros((rows, self.INDEX, 128), dtype=torch.float8_e4m3fn, device="cuda")
        self.index_factor = z(rows, self.INDEX)
        self.logits, self.tokens = z(rows, self.VOCAB).to(bf), torch.zeros(rows, dtype=torch.int64, device="cuda")
        self.uniforms, self.final = z(rows), z(3)
        self.counts = torch.zeros(3, dtype=torch.int32, device="cuda")
        self.weight, self.bias = (device(torch, rng.standard_normal(128), torch.float32) for _ in range(2))
        self.rotary = kvip_amd.Rotary(torch, rotary_dim=64, device="cuda")
        t = self.tables
        self.query_turn = kvip_amd.Rotary(torch, rotary_dim=64, device="cuda").bind(t.positions, self.query[..., 512:])
        self.store = kvip_amd.KvRowStore(torch, kv_cache=self.kv, rotary=self.rotary).bind(self.latent, self.rope, t.slots, t.positions)
        self.norm = kvip_amd.NormRotary(torch, rotary=kvip_amd.Rotary(torch, rotary_dim=64, layout="half", device="cuda"), dim=128,
                                        key_norm="layer")
        self.norm.bind(t.positions, self.index_q, self.index_k, key_weight=self.weight, key_bias=self.bias, query_out=self.index_codes,
                       query_scale=self.index_factor, slots=t.slots, key_cache=self.index_keys, key_scales=self.index_scales)
        self.attention = kvip_amd.ChunkAttention(torch, batch=3, heads=self.HEADS, max_tokens=rows, max_context=768, device="cuda")
        self.attention.bind(self.query, self.kv, t.block_table, t.lengths, t.cu_seqlens, steps=t.steps)
        self.history = kvip_amd.TokenHistory(torch, batch=3, vocab=self.VOCAB, device="cuda")
        self.temperature = device(torch, [0.8, 0.0, 1.1], torch.float32)
        self.penalty = device(torch, [1.2, 1.0, 1.5], torch.float32)
        self.sampler = kvip_amd.LogitProcessor(torch, batch=3, max_tokens=rows, vocab=self.VOCAB, device="cuda")
        self.sampler.bind(self.logits, t.cu_seqlens, temperature=self.temperature, history=self.history, repetition=self.penalty,
                          presence=self.temperature, tokens=self.tokens, visible=t.visible)
        self.verifier = kvip_amd.DraftVerifier(torch, batch=3, max_nodes=self.NODES, vocab=self.VOCAB, device="cuda")
        self.verifier.bind(self.sampler.probs, self.tokens, t.cu_seqlens, self.uniforms, self.final, steps=t.steps)

    def inputs(self, seed, counts):
        gen = self.torch.Generator(device="cuda").manual_seed(seed)
        for x in (self.latent, self.rope, self.query, self.index_q, self.index_k):
            x.copy_(self.torch.randn(x.shape, generator=gen, device="cuda"))
        self.logits.copy_(3 * self.torch.randn(self.logits.shape, generator=gen, device="cuda"))
        self.tokens.copy_(self.torch.randint(0, self.VOCAB, (self.ROWS,), generator=gen, device="cuda"))
        for x in (self.uniforms, self.final):
            x.copy_(self.torch.rand(x.shape, generator=gen, device="cuda"))
        self.counts.copy_(self.torch.tensor(counts, dtype=self.torch.int32))

    def layer(self):
        self.tables.extend(self.counts)
        self.query_turn()
        self.norm()
        self.store()
        return self.attention()

    def step(self):
        """A step of drafted chains: layer, sampler, verification; the kept tokens stay and are counted."""
        self.layer()
        self.sampler()
        tokens, kept, path = self.verifier()
        self.history.append(tokens, kept)
        self.tables.commit(kept, path)

    def state(self):
        t = self.tables
        out = [t.lengths, t.block_table, t.free_count, self.kv, self.index_keys.view(self.torch.uint8), self.index_scales,
               self.attention.output, self.index_codes.view(self.torch.uint8), self.index_factor, self.sampler.probs,
               self.verifier.out_tokens, self.verifier.kept, self.history.counts, self.history.seen]
        return [x.clone() for x in out]


def prompt_then_steps(torch, seed=40):
    p = Prompts(torch, seed)
    p.inputs(seed, [300, 1, 29])
    p.layer()
    p.tables.commit(p.counts)
    prompts = torch.randint(0, Prompts.VOCAB, (330,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    p.history.load(torch.arange(3, dtype=torch.int32, device="cuda"), prompts, p.tables.cu_seqlens, p.counts)
    return p, prompts


def test_a_prompt_and_steps_match(torch_gpu):
    torch = torch_gpu
    say("case prompt and steps")
    p, prompts = prompt_then_steps(torch)
    model = prompt.History(3, p.VOCAB)
    for b, (i, n) in enumerate(((0, 300), (300, 1), (301, 29))):
        model.load(b, prompts[i:i + n].tolist(), n)
    same_history(p.history, model)
    for seed, counts in ((41, [5, 6, 1]), (42, [1, 1, 4]), (43, [200, 1, 3])):
        p.inputs(seed, counts)
        if max(counts) <= p.NODES:
            bases = p.tables.lengths.tolist()
            p.layer()
        else:
            p.layer()
            bases = None
        lens, table, cu = p.tables.lengths.tolist(), p.tables.block_table.cpu().numpy(), p.tables.cu_seqlens.tolist()
        rows, got, q = p.kv.cpu().numpy().reshape(-1, ROW), host(p.attention.output), host(p.query)
        for b, n in enumerate(counts):
            key, value, _ = prompt.features(rows[[table[b, x // 128] * 128 + x % 128 for x in range(lens[b])]])
            for i in {0, n // 2, n - 1}:
                sees = lens[b] - n + i + 1
                want, _, bound, _ = prompt.attention(q[cu[b] + i], key[:sees], value[:sees], SCALE)
                assert np.all(np.abs(got[cu[b] + i] - want) <= bound + np.abs(want) * 2.0 ** -8), (b, i)
        if bases is None:
            p.tables.commit(p.counts)
            continue
        assert [x - n for x, n in zip(lens, counts)] == bases
        probs, x, names = host(p.sampler()), host(p.logits), p.tokens.tolist()
        for b, n in enumerate(counts):
            for i in range(n):
                way = [names[cu[b] + j] for j in range(1, i + 1)]
                z, slip, _ = prompt.logits(x[cu[b] + i], wrote=model.wrote[b], has=model.has[b], way=way,
                                           repetition=float(p.penalty[b]), presence=float(p.temperature[b]))
                want, bound = prompt.probabilities(z, slip, float(p.temperature[b]))
                if b == 1:
                    assert z[int(probs[cu[b] + i].argmax())] + slip.max() >= z.max() - slip.max()
                else:
                    assert np.all(np.abs(probs[cu[b] + i] - want) <= bound + want * 2.0 ** -24 + 2.0 ** -149)
        tokens, kept, path = p.verifier()
        p.history.append(tokens, kept)
        p.tables.commit(kept, path)
        for b in range(3):
            assert 1 <= int(kept[b]) <= counts[b]
            model.append(b, tokens[b, :int(kept[b])].tolist())
        same_history(p.history, model)
    for op in (p.tables, p.store, p.norm, p.attention, p.history, p.sampler, p.verifier):
        assert int(op.status.item()) == 0


def test_the_indexer_reads_what_the_norm_writes(torch_gpu):
    """Index queries and keys as they leave NormRotary go through PrefillIndexer: each row selects every row it sees (fewer
    than 2048)."""
    torch = torch_gpu
    say("case indexer after norm")
    p, _ = prompt_then_steps(torch, 44)
    p.inputs(45, [60, 9, 100])
    p.layer()
    t, n = p.tables, 169
    indexer = kvip_amd.PrefillIndexer(torch, max_rows=n, max_context=768, max_sequences=3, device="cuda", heads=p.INDEX)
    top = indexer(p.index_codes[:n], torch.ones((n, p.INDEX), device="cuda"), p.index_factor[:n].contiguous(), p.index_keys, p.index_scales,
                  t.cu_seqlens, t.lengths, t.block_table).cpu().numpy()
    lens, at = t.lengths.tolist(), 0
    for b, count in enumerate((60, 9, 100)):
        for i in range(count):
            sees = lens[b] - count + i + 1
            assert sorted(top[at + i][:sees].tolist()) == list(range(sees)) and np.all(top[at + i][sees:] == -1)
        at += count


def test_captured_steps_replay(torch_gpu):
    """A step captured once, replayed with other inputs and the program's own work between, against the same steps run
    eagerly."""
    torch = torch_gpu
    say("case captured steps")
    plan = [(50, [5, 6, 1]), (51, [1, 1, 4]), (52, [6, 1, 6]), (53, [2, 2, 2]), (54, [1, 6, 3])]
    eager, _ = prompt_then_steps(torch)
    want = []
    for seed, counts in plan:
        eager.inputs(seed, counts)
        eager.step()
        want.append(eager.state())
    p, _ = prompt_then_steps(torch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.step()
    for (seed, counts), expected in zip(plan, want):
        p.inputs(seed, counts)
        graph.replay()
        for a, b in zip(p.state(), expected):
            assert torch.equal(a, b), seed
        assert int(torch.ones(1000, device="cuda").sum().item()) == 1000
        torch.cuda.synchronize()


def test_calls_take_the_current_stream(torch_gpu):
    torch = torch_gpu
    say("case streams")
    side = torch.cuda.Stream()
    p, _ = prompt_then_steps(torch)
    p.inputs(60, [4, 5, 6])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        p.step()
        got = p.state()
    side.synchronize()
    q, _ = prompt_then_steps(torch)
    q.inputs(60, [4, 5, 6])
    q.step()
    for a, b in zip(got, q.state()):
        assert torch.equal(a, b)


def test_objects_run_side_by_side(torch_gpu):
    """Two objects of each kind on two streams at once: each has its own workspace."""
    torch = torch_gpu
    say("case side by side")
    pair = [prompt_then_steps(torch, seed)[0] for seed in (70, 71)]
    alone = []
    for seed in (70, 71):
        p = prompt_then_steps(torch, seed)[0]
        p.inputs(seed + 5, [6, 3, 5])
        p.step()
        alone.append(p.state())
    for p, seed in zip(pair, (70, 71)):
        p.inputs(seed + 5, [6, 3, 5])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pair]
    for p, stream in zip(pair, streams):
        with torch.cuda.stream(stream):
            p.step()
    torch.cuda.synchronize()
    for p, expected in zip(pair, alone):
        for a, b in zip(p.state(), expected):
            assert torch.equal(a, b)
