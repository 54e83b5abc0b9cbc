"""What the operators around a prompt chunk's layers (include/kvip_hip_prompt.h) owe their callers beyond ordinary inputs:
histories that only their bits speak for, tokens that tie, numbers at the ends of their range, calls that repeat
themselves, requests that claim the same rows. Values come from oracle/prompt.py or follow from the inputs."""
import math

import numpy as np
import pytest

import kvip_amd
from kvip_amd.runtime import abi
from oracle import prompt
from tests.test_gpu_draft import HALF_STEP, SCALE, device, dtype_of, host, say
from tests.test_gpu_prompt import LOWEST, Chunks, Sampling

pytestmark = pytest.mark.gpu


# --- logits ----------------------------------------------------------------------------------


@pytest.mark.parametrize("vocab,biases", [(60, 0), (700, 40), (9001, 300), (40000, 0)])
def test_counts_without_their_bit_are_not_read(torch_gpu, vocab, biases):
    """Counts of tokens that the request does not hold, next to tokens that it does, in the dense pass and in the lists; and a
    request that was cleared by its bits alone."""
    torch = torch_gpu
    say(f"case counts without bits vocab={vocab} biases={biases}")
    s = Sampling(torch, np.random.default_rng(vocab), [6, 1, 9, 2], vocab, "fp32", biases=biases)
    assert 0 < len(s.model.has[0]) < vocab
    s.history.seen[2] = 0
    s.model.wrote[2].clear()
    s.model.has[2].clear()
    counts, _ = s.model.arrays()
    for b, has in enumerate(s.model.has):
        others = np.setdiff1d(np.arange(vocab), list(has))
        counts[b, others] = 1 + others % 5
    s.history.counts.copy_(torch.from_numpy(counts))
    op = s.op()
    s.check(op())
    assert int(op.status.item()) == 0


def odd_reciprocals():
    """Numbers of 8 bits in 1..2 whose rounded reciprocal times themselves is not 1 in 32 bits."""
    r = (np.arange(129, 256) / 128).astype(np.float32)
    return r[r * (np.float32(1) / r) != 1]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("vocab", [700, 30000])
@pytest.mark.parametrize("listed", [None, "first", "second", "drafted"])
def test_the_first_of_equal_logits_wins(torch_gpu, dtype, vocab, listed):
    """A held token whose logit over the repetition penalty is exactly another's logit, whichever of them a bias of 0 or a
    draft names. Every number here is exact in 32 bits, so that there is one answer."""
    torch = torch_gpu
    say(f"case equal logits {dtype} vocab={vocab} listed={listed}")
    r = odd_reciprocals()[:30]
    n, first, second = len(r), 5, 600
    drafted = listed == "drafted"
    rows = 2 * n if drafted else n
    last = np.arange(1, rows, 2) if drafted else np.arange(n)  # the row of each request that is looked at
    x = np.full((rows, vocab), -9.0, np.float32)
    x[last, first], x[last, second] = r, 1.0
    history = kvip_amd.TokenHistory(torch, batch=n, vocab=vocab, device="cuda")
    tokens, visible = np.full(rows, 77), np.ones(rows, np.int64)
    kw = {}
    if drafted:  # row 1 comes behind the drafted token
        tokens[last], visible[last] = first, 3
        kw = dict(tokens=device(torch, tokens, torch.int64), visible=device(torch, visible, torch.int64))
    else:
        history.load(device(torch, range(n), torch.int32), torch.full((n,), first, dtype=torch.int64, device="cuda"),
                     device(torch, range(n + 1), torch.int32), device(torch, [1] * n, torch.int32))
    if listed in ("first", "second"):
        kw = dict(bias_tokens=torch.full((n, 1), first if listed == "first" else second, dtype=torch.int32, device="cuda"),
                  bias_values=torch.zeros((n, 1), device="cuda"))
    op = kvip_amd.LogitProcessor(torch, batch=n, max_tokens=rows, vocab=vocab, device="cuda")
    op.bind(device(torch, x, dtype_of(torch, dtype)), device(torch, np.arange(n + 1) * (rows // n), torch.int32), history=history,
            temperature=torch.zeros(n, device="cuda"), repetition=device(torch, r, torch.float32), **kw)
    got = host(op())[last]
    assert np.array_equal(got.argmax(1), np.full(n, first)) and np.all(np.count_nonzero(got, axis=1) == 1)
    assert int(op.status.item()) == 0


@pytest.mark.parametrize("vocab", [700, 30000])
def test_equal_tokens_get_equal_sums(torch_gpu, vocab):
    """Tokens of one logit, all held and written as often, of which a bias of 0 names some: the first wins, whether it is
    named or not, with penalties that no 32-bit number is."""
    torch = torch_gpu
    say(f"case equal sums vocab={vocab}")
    rng = np.random.default_rng(vocab)
    n = 64
    x = np.full((n, vocab), -30.0, np.float32)
    held = np.sort(np.stack([rng.permutation(vocab)[:6] for _ in range(n)]), axis=1)
    x[np.arange(n)[:, None], held] = rng.uniform(0.5, 9, (n, 1)).astype(np.float32)
    history = kvip_amd.TokenHistory(torch, batch=n, vocab=vocab, device="cuda")
    history.load(device(torch, range(n), torch.int32), device(torch, np.repeat(held, 3, axis=1).reshape(-1), torch.int64),
                 device(torch, np.arange(n + 1) * 18, torch.int32), torch.zeros(n, dtype=torch.int32, device="cuda"))
    numbers = {k: device(torch, rng.uniform(low, high, n), torch.float32) for k, low, high in
               (("repetition", 1.01, 1.9), ("presence", 0.01, 0.9), ("frequency", 0.01, 0.3))}
    for named in ((0,), (1, 3), (0, 1, 2, 3, 4, 5), ()):
        kw = {}
        if named:
            kw = dict(bias_tokens=device(torch, held[:, list(named)], torch.int32), bias_values=torch.zeros((n, len(named)), device="cuda"))
        op = kvip_amd.LogitProcessor(torch, batch=n, max_tokens=n, vocab=vocab, device="cuda")
        op.bind(device(torch, x, torch.float32), device(torch, range(n + 1), torch.int32), history=history,
                temperature=torch.zeros(n, device="cuda"), **numbers, **kw)
        got = host(op())
        assert np.array_equal(got.argmax(1), held[:, 0]) and np.all(np.count_nonzero(got, axis=1) == 1), named


@pytest.mark.parametrize("vocab,biases", [(20000, 4096), (140001, 2000), (3000, 600)])
def test_tokens_named_twice_repeat_themselves(torch_gpu, vocab, biases):
    """Lists whose entries meet in pairs, from other threads and other waves: every call gives the same bits."""
    torch = torch_gpu
    say(f"case named twice vocab={vocab} biases={biases}")
    rng = np.random.default_rng(biases)
    s = Sampling(torch, rng, [1] * 40, vocab, "fp32", biases=biases)
    s.numbers["temperature"][:] = 1.5
    for b in range(40):
        s.names[b, :biases // 2] = rng.permutation(vocab)[:biases // 2]
        s.names[b, biases // 2:] = np.roll(s.names[b, :biases // 2], 1 + 64 * b)
    op = s.op()
    first = op().clone()
    for _ in range(60):
        assert torch.equal(op(), first)
    s.check(first)


def test_one_token_of_many_named_twice(torch_gpu):
    """Lists of 4096 different tokens but for one pair, or one token named by drafts and biases alike."""
    torch = torch_gpu
    say("case one pair")
    rng = np.random.default_rng(21)
    s = Sampling(torch, rng, [1, 30], 30000, "fp32", biases=4096, masked=True)
    s.numbers["temperature"][:] = 0.9
    s.allowed[:, 0] |= 1
    for b in range(2):
        s.names[b] = rng.permutation(30000)[:4096]
    for pair in ((0, 1), (4095, 0), (511, 512), (100, 4000)):
        names = s.names.copy()
        s.names[:, pair[1]] = s.names[:, pair[0]]
        op = s.op()
        s.check(op())
        s.names = names
    s.names[:, 70], s.names[:, 3000] = s.tokens[s.cu[:-1] + [0, 5]], s.tokens[s.cu[:-1] + [0, 5]]
    op = s.op()
    s.check(op())
    assert int(op.status.item()) == 0


@pytest.mark.parametrize("vocab", [40, 30000])
@pytest.mark.parametrize("listed", [False, True])
def test_infinite_logits_take_the_row_at_any_temperature(torch_gpu, vocab, listed):
    """Tokens at +infinity share their row, others get nothing, under temperatures up to infinity."""
    torch = torch_gpu
    say(f"case infinite logits vocab={vocab} listed={listed}")
    t = device(torch, [math.inf, 3.4e38, 1e37, 1e30, 1.0, 1e-30, 1e-42, 0.0], torch.float32)
    x = torch.randn((8, vocab), generator=torch.Generator().manual_seed(2)).cuda()
    kw = {}
    if listed:
        kw = dict(bias_tokens=device(torch, [[7, 30]] * 8, torch.int32), bias_values=torch.full((8, 2), math.inf, device="cuda"))
    else:
        x[:, 7] = x[:, 30] = math.inf
    op = kvip_amd.LogitProcessor(torch, batch=8, max_tokens=8, vocab=vocab, device="cuda")
    got = host(op.bind(x, device(torch, range(9), torch.int32), temperature=t, **kw)())
    want = np.zeros((8, vocab))
    want[:, 7] = want[:, 30] = 0.5
    want[7, 7], want[7, 30] = 1.0, 0.0
    assert np.array_equal(got, want) and int(op.status.item()) == 0


# --- norm and rotation -----------------------------------------------------------------------


@pytest.mark.parametrize("exponent", [0, 3, -40, 90, -105, -124])
@pytest.mark.parametrize("half", [False, True])
def test_codes_of_features_half_way_between_two(torch_gpu, exponent, half):
    """Features that are exactly half-way between two codes times the head's scale go to the even one, whatever the scale.
    Every number is exact in 32 bits, so that there is one answer."""
    torch = torch_gpu
    say(f"case half-way codes 2^{exponent} half={half}")
    scales = (np.arange(128, 256) / 128).astype(np.float32)
    scales = scales[scales * np.float32(448) / np.float32(448) == scales]
    values = np.concatenate([np.arange(17, 32, 2) * 2.0 ** k for k in (-3, 0, 3)] + [[448.0, 0.0]])
    heads = np.zeros((len(scales), 128))
    heads[:, :len(values)] = values
    heads[:, 64:64 + len(values)] = -values
    x = (heads * scales[:, None] * 2.0 ** exponent).astype(np.float32)
    assert np.array_equal(x.astype(np.float64), heads * scales[:, None] * 2.0 ** exponent)
    want, scale = prompt.codes(heads)
    assert np.all(scale == 1)
    n = len(scales)
    turn = kvip_amd.Rotary(torch, rotary_dim=64, layout="half" if half else "interleaved", device="cuda")
    op = kvip_amd.NormRotary(torch, rotary=turn, dim=128)
    codes, factor = torch.zeros((n, 1, 128), dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros((n, 1), device="cuda")
    pages, page_scales = torch.zeros((1, 128, 128), dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros((1, 128), device="cuda")
    heads = device(torch, x[:, None], torch.float32)
    op.bind(torch.zeros(n, dtype=torch.int64, device="cuda"), heads, heads.clone(), query_out=codes, query_scale=factor,
            slots=torch.arange(n, device="cuda"), key_cache=pages, key_scales=page_scales)()
    for got, s in ((codes[:, 0], factor[:, 0]), (pages[0, :n], page_scales[0, :n])):
        assert np.array_equal(host(s), scales * 2.0 ** exponent)
        assert np.array_equal(host(got.float()), want)
    assert int(op.status.item()) == 0


# --- attention -------------------------------------------------------------------------------


@pytest.mark.parametrize("heads,counts,contexts,cu", [
    (128, [1000, 0, 900, 0, 1000], [1000, 0, 600, 0, 100], [0, 1000, 100, 1000, 100, 1100]),
    (16, [100, 0, 90, 0, 90, 0, 100], [9000, 0, 9000, 0, 9000, 0, 8000], [0, 100, 10, 100, 10, 100, 10, 110])])
def test_rows_that_several_requests_claim_are_the_first_ones(torch_gpu, heads, counts, contexts, cu):
    """cu_seqlens that fall: every row is written, by the first request that has it, and the status says so."""
    torch = torch_gpu
    say(f"case claimed rows heads={heads} cu={cu}")
    step = Chunks(torch, np.random.default_rng(heads), counts, contexts, heads)
    step.cu, step.tokens = np.asarray(cu, np.int32), cu[-1] + 5
    step.query = step.query[:step.tokens].contiguous()
    op = step.run()
    got, lse, q = host(op()), host(op.lse), step.query.double().numpy()
    assert int(op.status.item()) == abi.STATUS_BAD_LENGTH
    last, shared = len(counts) - 1, max(cu[:-1])
    for b, rows in ((0, (0, cu[2] - 1, cu[2], cu[1] - 1)), (last, (shared, shared + 3, cu[-1] - 1))):
        key, value, odd = prompt.features(step.rows[[step.slot(b, p) for p in range(step.lens[b])]])
        assert not odd.any()
        for row in rows:
            sees = step.lens[b] - (cu[b + 1] - row) + 1
            want, want_lse, bound, lse_bound = prompt.attention(q[row], key[:sees], value[:sees], SCALE)
            assert np.all(np.abs(got[row] - want) <= bound + np.abs(want) * 2.0 ** -8), (b, row)
            assert np.all(np.abs(lse[row] - want_lse) <= lse_bound), (b, row)
    assert not np.any(np.all(got[:cu[-1]] == 3.0, axis=(1, 2)))
    assert np.all(got[cu[-1]:] == 3.0) and np.all(lse[cu[-1]:] == 3.0)


def test_a_long_request_keeps_its_sums(torch_gpu):
    """2^20 rows, one page over and over: that page's attention, with log(2^13) more in the log-sum-exp.

    The plan cuts a lone long request into 32 segments of 1024 tiles of 32 rows. A sum of probabilities is 16 terms per tile and
    lane, then 1024 additions, then 2 lanes and 32 parts, each off by 2^-24 of the sum at most: (16 + 1024 + 33) 2^-24 <
    2^-13.8. An output sum is 2 matrix products per tile with at most 16 roundings each: 2^15 2^-24 = 2^-9 of the
    sum of magnitudes; features are positive here, so that this is the output's own size."""
    torch = torch_gpu
    say("case long sums")
    rng = np.random.default_rng(31)
    step = Chunks(torch, rng, [1], [127], 16, spare=0)
    step.rows[:, :512] &= 0x7F  # positive features
    key, value, odd = prompt.features(step.rows)
    assert not odd.any() and len(step.rows) == 128 and np.all(value >= 0)
    length = 1 << 20
    op = kvip_amd.ChunkAttention(torch, batch=1, heads=16, max_tokens=71, max_context=length, device="cuda", output_dtype=torch.float32, lse=True)
    op.bind(step.query.cuda(), torch.from_numpy(step.rows).cuda().view(1, 128, -1), torch.zeros((1, length // 128), dtype=torch.int32, device="cuda"),
            device(torch, [length], torch.int32), device(torch, [0, 1], torch.int32))
    got, lse = host(op())[0], host(op.lse)[0]
    # Each probability's rounding to fp16 is in the page's own bound: it is the same one in every repetition, 2^-36 of the largest
    # feature per row among the smallest.
    want, want_lse, bound, lse_bound = prompt.attention(step.query.double().numpy()[0], key, value, SCALE)
    assert np.all(np.abs(got - want) <= bound + want * (2.0 ** -9 + 2.0 ** -13.8))
    assert np.all(np.abs(lse - (want_lse + math.log(length // 128))) <= lse_bound + 2.0 ** -13.8 + 20 * 2.0 ** -23)
    assert int(op.status.item()) == 0


@pytest.mark.parametrize("power", [-60, -112, -120, -126, -133, 112, 118])
@pytest.mark.parametrize("output", ["fp32", "bf16"])
@pytest.mark.parametrize("heads,counts,contexts", [(16, [70, 3], [900, 40]), (4, [20, 50], [9000, 10])])
def test_chunk_attention_of_rows_near_the_ends_of_the_range(torch_gpu, power, output, heads, counts, contexts):
    """Rows whose features come near the smallest normal number, and pass it, or near the largest (under queries that keep the
    logits ordinary): outputs as exact as elsewhere, but
    for a step of 2^-149 (bf16: 2^-133) at each of two roundings."""
    torch = torch_gpu
    say(f"case chunk rows of 2^{power} {output} counts={counts}")
    step = Chunks(torch, np.random.default_rng(heads), counts, contexts, heads)
    scales = step.rows[:, 640:656].copy().view("<f4")
    used = np.isfinite(scales).all(1)
    scales[used] = 2.0 ** power
    step.rows[:, 640:656] = scales.astype("<f4").view(np.uint8)
    step.rows[used, 512:640] = 0  # rotary features
    if power > 0:
        step.query = (step.query.float() * 2.0 ** -power).to(torch.bfloat16)
    op = step.run(output=output)
    got, q = host(op()), step.query.double().numpy()
    for b, n in enumerate(counts):
        key, value, odd = prompt.features(step.rows[[step.slot(b, p) for p in range(step.lens[b])]])
        assert not odd.any()
        for i in sorted({0, n // 2, n - 1}):
            row, sees = step.cu[b] + i, step.lens[b] - n + i + 1
            want, _, bound, _ = prompt.attention(q[row], key[:sees], value[:sees], SCALE)
            bound = bound + np.abs(want) * HALF_STEP[output] + 2 * LOWEST[output] + 2.0 ** -148
            assert np.all(np.abs(got[row] - want) <= bound), (b, i, float((np.abs(got[row] - want) / bound).max()))
            assert np.abs(want).max() > 2.0 ** (power - 3)


def test_chunk_attention_of_nothing_but_nan(torch_gpu):
    """Long contexts whose rotary features are all NaN, or NaN in one row of the first segment, cut into many parts."""
    torch = torch_gpu
    say("case chunk NaN parts")
    step = Chunks(torch, np.random.default_rng(17), [2, 3], [9000, 9000], 4)
    used = [step.slot(0, p) for p in range(step.lens[0])]
    step.rows[used, 512:640] = 0xFF
    step.rows[step.slot(1, 5), 512:514] = [0xC0, 0x7F]
    op = step.run()
    got, lse = host(op()), host(op.lse)
    assert np.all(np.isnan(got[:5])) and np.all(np.isnan(lse[:5])) and int(op.status.item()) == 0
