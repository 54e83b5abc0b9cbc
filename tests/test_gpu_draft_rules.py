"""GPU tests of what the drafted round's operators promise at the edges of their rules: steps without
parents, requests that got no pages, targets whose support was drafted whole, workspaces of several
shapes, latents and scales at the ends of their range. Against oracle/draft.py, with the bounds of
tests/test_gpu_draft.py."""
import math

import numpy as np
import pytest

import kvip_amd
from kvip_amd.runtime import abi
from oracle import draft
from tests.test_gpu_draft import (HALF_STEP, ROW, SCALE, Round, Step, check_verify, device, dtype_of, host,
                                  random_parents, run_verify, same_tables, say, softmax_rows, verify_case)

pytestmark = pytest.mark.gpu


# --- steps without parents -------------------------------------------------------------------


def same(tensor, values, dtype=np.int64):
    return np.array_equal(tensor.cpu().numpy(), np.asarray(values, dtype).view(np.int64))


@pytest.mark.parametrize("batch,blocks,pages,rows,most", [(1, 1, 1, 1, 2), (3, 5, 9, 40, 20), (70, 9, 200, 900, 14),
                                                          (257, 33, 3000, 20000, 200)])
def test_visibility_follows_every_extend(torch_gpu, batch, blocks, pages, rows, most):
    """Steps with and without parents in turn on one object; some requests without tokens, some refused."""
    torch = torch_gpu
    rng = np.random.default_rng(batch + rows)
    say(f"case visibility batch={batch} rows={rows}")
    op = kvip_amd.PageTables(torch, batch=batch, max_context=blocks * 128, num_blocks=pages, max_tokens=rows, device="cuda")
    model = draft.Tables(batch, blocks, pages, rows)
    for step in range(6):
        counts = rng.integers(0, most, batch)
        counts[rng.random(batch) < 0.2] = 0
        parents = random_parents(rng, counts, rows) if step % 3 == 1 and counts.max() <= 64 else None
        op.extend(device(torch, counts, torch.int32), None if parents is None else device(torch, parents, torch.int32))
        want = model.extend(counts.tolist(), parents)
        assert same(op.visible, want[3], np.uint64), step
        assert same(op.slots, want[1]) and same(op.positions, want[2]), step
        same_tables(op, model)
        op.truncate(device(torch, np.minimum(model.lengths, blocks * 40), torch.int32))
        model.truncate([min(x, blocks * 40) for x in model.lengths])


def chain_or_tree_step(r, model, counts, parents):
    """One step of a Round's tables, store and attention, the attention's rows against the restatement."""
    torch = r.torch
    _, _, _, visible, status = model.extend(counts, None if parents is None else parents.tolist())
    assert status == 0
    r.tables.extend(r.counts, None if parents is None else device(torch, parents, torch.int32))
    r.rotary()
    r.store()
    got, rows = host(r.attention()), r.kv.cpu().numpy().reshape(-1, ROW)
    q, at = host(r.query), 0
    for b, n in enumerate(counts):
        held = rows[[model.pages[b][p // 128] * 128 + p % 128 for p in range(model.lengths[b])]]
        for i in range(n):
            sees = np.ones(len(held), bool)
            sees[len(held) - n:] = [bool(visible[at + i] >> j & 1) for j in range(n)]
            want, _, bound, _ = draft.tree_attention(q[at + i], held, sees, SCALE)
            assert np.all(np.abs(got[at + i] - want) <= bound + np.abs(want) * HALF_STEP["bf16"]), (b, i)
        at += n


def test_a_bound_attention_takes_trees_and_chains_in_turn(torch_gpu):
    """The attention stays bound to the tables' visibility; a step without drafts (one token), a chain and a tree
    follow one another."""
    torch = torch_gpu
    say("case trees and chains in turn")
    r, model = Round(torch, 11), draft.Tables(3, 8, 40, 25)
    plan = [([1, 1, 1], False), ([7, 5, 6], True), ([4, 6, 7], False), ([1, 0, 1], False), ([7, 2, 3], True), ([7, 7, 7], False)]
    for seed, (counts, tree) in enumerate(plan):
        r.inputs(seed, counts)
        parents = r.parents.cpu().numpy() if tree else None
        chain_or_tree_step(r, model, counts, parents)
        kept = [n - n // 3 for n in counts]
        r.tables.commit(device(torch, kept, torch.int32))
        model.commit(kept)
        same_tables(r.tables, model)
    for op in (r.tables, r.store, r.attention):
        assert int(op.status.item()) == 0


# --- requests that got no pages --------------------------------------------------------------


def random_rows(rng, count):
    """uint8 [count, 656]: rows of N(0, 1) latents and rotary features."""
    rows = np.zeros((count, ROW), np.uint8)
    codes, scales = draft.stored_rows(rng.standard_normal((count, 512)).astype(np.float32))
    rows[:, :512], rows[:, 640:656] = codes, scales.view(np.uint8)
    rope = rng.standard_normal((count, 64)).astype(np.float32)
    rows[:, 512:640] = (rope.view(np.uint32) >> 16).astype("<u2").view(np.uint8)
    return rows


def test_a_refused_request_answers_nothing(torch_gpu):
    """A request that gets no page keeps its length and its rows of the step; nothing of it is attended or verified,
    the others go on, and so does it once there are pages."""
    torch = torch_gpu
    say("case refused request")
    r, rng = Round(torch, 21), np.random.default_rng(21)
    t = r.tables
    r.attention.bind(r.query, r.kv, t.block_table, t.lengths, t.cu_seqlens, t.visible, steps=t.steps)
    r.verifier.bind(r.probs, r.tokens, t.cu_seqlens, r.uniforms, r.final, parents=r.parents, steps=t.steps)
    r.kv.copy_(torch.from_numpy(random_rows(rng, 40 * 128)).view(40, 128, ROW))
    for counts in [[0, 25, 0]] * 5 + [[21, 0, 0]] * 2 + [[0, 0, 21]] * 2:
        t.extend(device(torch, counts, torch.int32))
        t.commit(device(torch, counts, torch.int32))
    assert t.lengths.tolist() == [42, 125, 42] and int(t.status.item()) == 0
    counts, pages = [6, 7, 5], t.free_count.clone()
    for seed, there in ((3, False), (4, True)):
        t.free_count.copy_(pages if there else torch.zeros_like(pages))  # the other pages are someone else's
        t.status.zero_()
        r.inputs(seed, counts)
        bases = t.lengths.tolist()
        r.step()
        table, kept = t.block_table.cpu().numpy(), r.verifier.kept.tolist()
        assert int(t.status.item()) == (0 if there else abi.STATUS_NO_PAGE)
        assert t.lengths.tolist() == [n + k for n, k in zip(bases, kept)]
        at, probs = 0, host(r.probs)
        for b, n in enumerate(counts):
            s = slice(at, at + n)
            at += n
            if b == 1 and not there:
                assert kept[b] == 0 and set(r.verifier.out_tokens[b].tolist()) == set(r.verifier.path[b].tolist()) == {-1}
                assert not r.attention.output[s].any() and t.slots[s].tolist() == [-1] * n
                continue
            walk, out = draft.verify(probs[s], r.tokens[s].tolist(), r.parents[s].tolist(), None, r.uniforms[s].tolist(),
                                     float(r.final[b]))
            assert r.verifier.path[b].tolist()[:kept[b]] == walk and r.verifier.out_tokens[b].tolist()[:kept[b]] == out
            # The first token sees the rows before it, which the step leaves where they were, and itself.
            rows = r.kv.cpu().numpy().reshape(-1, ROW)[[table[b, p // 128] * 128 + p % 128 for p in range(bases[b] + 1)]]
            want, _, bound, _ = draft.tree_attention(host(r.query)[s][0], rows, np.ones(len(rows), bool), SCALE)
            assert np.all(np.abs(host(r.attention.output)[s][0] - want) <= bound + np.abs(want) * HALF_STEP["bf16"])
    for op in (r.store, r.attention, r.verifier):
        assert int(op.status.item()) == 0


@pytest.mark.parametrize("heads,counts,contexts,steps", [
    (16, [3, 2, 4], [200, 300, 0], [3, 0, 4]), (16, [64, 2], [1000, 40], [0, 2]), (128, [12, 5, 9], [4000, 900, 20], [12, 0, 9]),
    (40, [7, 1], [20000, 30000], [7, 0]), (8, [1] * 90, [(53 * i) % 900 for i in range(90)], [i % 3 and 1 for i in range(90)])])
def test_attention_of_refused_requests_is_zero(torch_gpu, heads, counts, contexts, steps):
    torch = torch_gpu
    say(f"case refused attention heads={heads} counts={counts[:5]}")
    step = Step(torch, np.random.default_rng(heads), counts, contexts, heads)
    op = step.run()
    query, kv, table, lens, cu, visible = op._bound[:6]
    op.bind(query, kv, table, lens, cu, visible, steps=device(torch, steps, torch.int32))
    step.check(op, only=[b for b, n in enumerate(steps) if n])
    for b, n in enumerate(steps):
        if n == 0:
            rows = slice(int(step.cu[b]), int(step.cu[b + 1]))
            assert not op.output[rows].any() and bool((op.lse[rows] == -math.inf).all()), b
    assert int(op.status.item()) == 0
    again = kvip_amd.tree_attention(query, kv, table, lens, cu, visible, max_nodes=max(counts), steps=device(torch, steps, torch.int32))
    assert torch.equal(again[:int(step.cu[-1])], op.output[:int(step.cu[-1])])
    for bad in (device(torch, steps, torch.int64), device(torch, steps[:-1], torch.int32), device(torch, steps, torch.int32).cpu()):
        with pytest.raises(ValueError):
            op.bind(query, kv, table, lens, cu, visible, steps=bad)


@pytest.mark.parametrize("drafted", ["tree", "draft"])
def test_verification_of_refused_requests_keeps_nothing(torch_gpu, drafted):
    torch = torch_gpu
    say(f"case refused verification {drafted}")
    rng = np.random.default_rng(5)
    counts, steps = [4, 5, 0, 6], [4, 0, 0, 6]
    case = verify_case(torch, rng, counts, 9001, drafted, "fp32")
    op = run_verify(torch, case, nodes=6, vocab=9001)
    check_verify(case, op, nodes=6)
    all_tokens, all_kept, all_path = (x.clone() for x in (op.out_tokens, op.kept, op.path))
    probs, q, tokens, cu, parents, uniforms, final = op._bound[:7]
    named = dict(parents=parents, draft_probs=q)
    op.bind(probs, tokens, cu, uniforms, final, steps=device(torch, steps, torch.int32), **named)()
    assert int(op.kept[1]) == 0 and bool((op.out_tokens[1] == -1).all()) and bool((op.path[1] == -1).all())
    for b in (0, 2, 3):
        assert torch.equal(op.out_tokens[b], all_tokens[b]) and torch.equal(op.path[b], all_path[b])
        assert op.kept[b] == all_kept[b]
    assert int(op.status.item()) == 0
    for bad in (device(torch, steps, torch.int64), device(torch, steps[:-1], torch.int32), device(torch, steps, torch.int32).cpu()):
        with pytest.raises(ValueError):
            op.bind(probs, tokens, cu, uniforms, final, steps=bad, **named)


def test_a_captured_round_with_refusals_replays(torch_gpu):
    """A captured round whose pages run out on some replays, against a second engine that runs every round eagerly."""
    torch = torch_gpu
    say("case captured refusals")
    engines = [Round(torch, 25), Round(torch, 25)]
    for r in engines:
        t = r.tables
        r.attention.bind(r.query, r.kv, t.block_table, t.lengths, t.cu_seqlens, t.visible, steps=t.steps)
        r.verifier.bind(r.probs, r.tokens, t.cu_seqlens, r.uniforms, r.final, parents=r.parents, steps=t.steps)
    eager, graphed = engines
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for r in engines:
            for _ in range(5):
                r.tables.extend(device(torch, [0, 25, 0], torch.int32))
                r.tables.commit(device(torch, [0, 25, 0], torch.int32))
            r.inputs(0, [3, 2, 4])
            r.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        graphed.step()
    refused = 0
    for seed in range(1, 9):
        counts = [int(x) for x in np.random.default_rng(seed).integers(1, 8, 3)]
        pages = eager.tables.free_count.clone()
        for r in engines:
            r.inputs(seed, counts)
            if seed % 3:
                r.tables.free_count.zero_()
            r.tables.status.zero_()
        bases = eager.tables.lengths.tolist()
        eager.step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.state(), graphed.state()):
            assert torch.equal(a, b), seed
        refused += sum(k == 0 for k in graphed.verifier.kept.tolist())
        assert graphed.tables.lengths.tolist() == [n + k for n, k in zip(bases, graphed.verifier.kept.tolist())]
        if seed % 3:
            for r in engines:
                r.tables.free_count.add_(pages)
        if seed == 4:  # back to the edge of a page, to be refused again
            for r in engines:
                r.tables.truncate(device(torch, [0, 127, 0], torch.int32))
    assert refused > 0


# --- targets whose support was drafted whole --------------------------------------------------


def one_row(torch, weights, tokens, parents, dtype, vocab, u, final, draft_row=None):
    """A case of one request per entry of `u` whose rows all have the same target."""
    t, n = dtype_of(torch, dtype), len(tokens)
    probs = torch.zeros((len(u) * n, vocab), dtype=t, device="cuda")
    for v, x in weights.items():
        probs[:, v] = x
    q = None
    if draft_row is not None:
        q = torch.zeros_like(probs)
        for v, x in draft_row.items():
            q[:, v] = x
    uniforms = np.zeros((len(u), n), np.float32)
    uniforms[:, 0] = u
    return dict(probs=probs, tokens=np.tile(tokens, len(u)), parents=None if parents is None else np.tile(np.int32(parents), len(u)),
                draft=q, cu=np.arange(len(u) + 1) * n, uniforms=uniforms.reshape(-1), final=np.float32(final))


@pytest.mark.parametrize("dtype,vocab", [("bf16", 2), ("bf16", 5000), ("fp32", 40000), ("fp16", 9001)])
def test_children_that_are_the_whole_support(torch_gpu, dtype, vocab):
    """bf16(0.1) + bf16(0.9) is 0.9985: a number above it falls to the last child with a weight, not to no token."""
    torch = torch_gpu
    say(f"case whole support {dtype} {vocab}")
    last = vocab - 1
    u = [0.0, 0.05, 0.1005, 0.5, 0.99, 0.999, 1 - 2.0 ** -24]
    for tokens, parents in (([0, 0, last], [-1, 0, 0]), ([0, last, 0], [-1, 0, 0]), ([0, 0, last, 0], [-1, 0, 0, 0])):
        case = one_row(torch, {0: 0.1, last: 0.9}, tokens, parents, dtype, vocab, u, np.linspace(0, 0.99, len(u)))
        case["probs"] *= 0.995  # fp32 and fp16 come short too
        op = run_verify(torch, case, nodes=len(tokens), vocab=vocab)
        check_verify(case, op, nodes=len(tokens))
        assert int(op.status.item()) == 0 and bool((op.out_tokens[:, 0] >= 0).all())
        first = op.out_tokens[:, 0].tolist()
        assert first[-1] == (last if tokens[1] == 0 else 0) and set(first) == {0, last}
    # A chain's only child is the whole target; a child without a weight is not drawn either.
    case = one_row(torch, {last: 0.998}, [0, last], None, dtype, vocab, u, np.linspace(0, 0.99, len(u)))
    op = run_verify(torch, case, nodes=2, vocab=vocab)
    check_verify(case, op, nodes=2)
    assert op.out_tokens[:, 0].tolist() == [last] * len(u) and op.kept.tolist() == [2] * 5 + [1, 1]
    if vocab > 2:
        case = one_row(torch, {last: 0.998}, [0, last, 1], [-1, 0, 0], dtype, vocab, u, np.linspace(0, 0.99, len(u)))
        op = run_verify(torch, case, nodes=3, vocab=vocab)
        check_verify(case, op, nodes=3)
        assert op.out_tokens[:, 0].tolist() == [last] * len(u) and int(op.status.item()) == 0


@pytest.mark.parametrize("dtype,vocab", [("bf16", 2), ("bf16", 5000), ("fp32", 40000), ("fp16", 9001)])
def test_a_refusal_that_leaves_no_residual(torch_gpu, dtype, vocab):
    """A drafted token whose target is a rounding step below its draft is refused now and then, and
    max(p - q, 0) is 0 everywhere: the target itself is drawn from."""
    torch = torch_gpu
    say(f"case no residual {dtype} {vocab}")
    last, final = vocab - 1, [0.0, 0.1, 0.4, 0.6, 0.9, 1 - 2.0 ** -24]
    u = [1 - 2.0 ** -24] * len(final)
    case = one_row(torch, {0: 0.5, last: 0.5 - 2.0 ** -9}, [0, last], None, dtype, vocab, u, final, {0: 0.5, last: 0.5})
    op = run_verify(torch, case, nodes=2, vocab=vocab)
    for _ in range(2):
        check_verify(case, op, nodes=2)
        assert op.kept.tolist() == [1] * len(final) and op.out_tokens[:, 0].tolist() == [0] * 3 + [last] * 3
    assert int(op.status.item()) == 0
    if vocab < 4:
        return
    rng = np.random.default_rng(vocab)  # a target of many tokens, each at most its draft
    p = softmax_rows(rng, 2, vocab, sharp=1.0)[:1]
    case["probs"].copy_(torch.from_numpy(p))
    case["draft"].copy_(case["probs"])
    token = int(p.argmax())
    case["tokens"][1::2] = token
    case["draft"][:, token] *= 1.25
    op = run_verify(torch, case, nodes=2, vocab=vocab)
    check_verify(case, op, nodes=2)
    assert op.kept.tolist() == [1] * len(final) and int(op.status.item()) == 0


def test_rows_without_any_weight_still_have_no_token(torch_gpu):
    torch = torch_gpu
    say("case no weight at all")
    for weights, draft_row in (({}, None), ({}, {0: 1.0}), ({0: -1.0, 7: float("nan")}, None), ({0: -1.0}, {0: 1.0, 7: 0.5}),
                               ({0: float("inf")}, {0: 1.0, 3: 1.0})):
        tokens, parents = ([0, 3], None) if draft_row else ([0, 3, 7], [-1, 0, 0])
        case = one_row(torch, weights, tokens, parents, "fp32", 5000, [0.0, 0.7], [0.0, 0.7], draft_row)
        op = run_verify(torch, case, nodes=len(tokens), vocab=5000)
        check_verify(case, op, nodes=len(tokens))
        assert op.out_tokens[:, 0].tolist() == [-1, -1] and int(op.status.item()) == abi.STATUS_BAD_PROBS


# --- one workspace, several shapes ------------------------------------------------------------


def test_a_workspace_serves_calls_of_other_shapes(torch_gpu):
    """One buffer, cleared once and large enough for each, under calls of different batches and vocabularies."""
    torch = torch_gpu
    say("case shared workspace")
    rng = np.random.default_rng(31)
    shapes = [(3, 40000), (40, 300), (20, 9001), (1, 100003), (200, 5000)]
    made = []
    for batch, vocab in shapes:
        case = verify_case(torch, rng, [3] * batch, vocab, "chain", "bf16")
        made.append((case, run_verify(torch, case, nodes=3, vocab=vocab)))
    words = max(op.workspace.numel() for _, op in made)
    shared = torch.zeros(words, dtype=torch.int64, device="cuda")
    for _, op in made:
        op.args.workspace = shared.data_ptr()
    for k in (0, 1, 2, 1, 3, 4, 0, 2, 4, 1):
        case, op = made[k]
        op.out_tokens.fill_(-9)
        check_verify(case, op, nodes=3)
        assert int(op.status.item()) == 0


# --- latents at the ends of their range -------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_latents_below_and_past_the_range(torch_gpu, dtype):
    """Groups whose largest magnitude over 448 is 0 in 32 bits are zeros with scale 1, not 0 / 0; a NaN stays in its
    feature, an infinity makes its scale infinite and itself a NaN; all as the restatement has them."""
    torch = torch_gpu
    say(f"case latents at the ends {dtype}")
    rng = np.random.default_rng(7)
    t = dtype_of(torch, dtype)
    tops = [1e-45, 1e-43, 3.1e-43, 3.2e-43, 1e-41, 1e-38, 1e-30, 6e-8, 1e-7, 1.0, 6e4, 3e38]
    x = rng.uniform(-1, 1, (len(tops) + 3, 512)).astype(np.float32)
    for i, top in enumerate(tops):
        x[i] *= np.float32(0.5 * top)
        x[i, ::128] = np.float32(top)
        x[i, 1::128] = 0.0
    x[-3, 5], x[-3, 200:384] = np.nan, np.nan
    x[-2, 130], x[-2, 131] = np.inf, np.nan
    x[-1, 400] = -np.inf
    latent = torch.from_numpy(x).to(t).cuda()
    rope = torch.zeros((len(x), 64), dtype=t, device="cuda")
    kv = torch.zeros((1, 128, ROW), dtype=torch.uint8, device="cuda")
    op = kvip_amd.KvRowStore(torch, kv_cache=kv)
    op.bind(latent, rope, torch.arange(len(x), device="cuda"))()
    values = latent.float().cpu().numpy()
    codes, scales = draft.stored_rows(values)
    got = kv[0, :len(x)].cpu().numpy()
    assert np.array_equal(got[:, 640:656].copy().view("<f4"), scales)
    none = (codes & 127) == 127
    assert np.array_equal((got[:, :512] & 127) == 127, none) and np.array_equal(got[:, :512][~none], codes[~none])
    finite = np.isfinite(values).all(1)
    assert not none[finite].any() and none[~finite].any(1).all()
    assert int(op.status.item()) == 0


# --- scales that are not finite ---------------------------------------------------------------


@pytest.mark.parametrize("heads,counts,contexts,at", [
    (16, [3, 2, 1], [300, 200, 90], [10, 40]), (128, [2, 1, 3], [700, 500, 40], [600, 3]), (16, [1, 1, 1], [127, 64, 31], [0, 40]),
    (40, [7, 5, 2], [20000, 9000, 300], [12000, 8900]), (8, [4] * 60, [400] * 60, [100, 399])])
def test_a_seen_scale_that_is_not_finite(torch_gpu, heads, counts, contexts, at):
    """Rows before the step, which every token sees: the first request holds an infinite scale, the second a
    negative one, and each token and head of theirs is NaN as a whole, whatever sign its products have."""
    say(f"case infinite scale heads={heads} counts={counts[:3]} contexts={contexts[:3]}")
    step = Step(torch_gpu, np.random.default_rng(heads + contexts[0]), counts, contexts, heads)
    scales = step.rows[:, 640:656].copy().view("<f4")
    scales[step.slot(0, at[0]), 1] = np.inf
    scales[step.slot(1, at[1]), 3] = -np.inf
    step.rows[:, 640:656] = scales.view(np.uint8)
    for output in ("bf16", "fp32"):
        op = step.run(output=output)
        step.check(op, output=output, only=range(2, len(counts)))
        bad = slice(0, int(step.cu[2]))
        assert bool(op.output[bad].isnan().all()) and bool(op.lse[bad].isnan().all())
        assert int(op.status.item()) == 0


# --- rows of the tables' caches ---------------------------------------------------------------


def test_caches_whose_rows_overlap_are_refused(torch_gpu):
    torch = torch_gpu
    make = dict(batch=2, max_context=512, num_blocks=4, max_tokens=16, device="cuda")
    flat = torch.zeros(8 * 128 * 16, dtype=torch.uint8, device="cuda")
    one = flat[:128 * 16].view(1, 128, 16)
    for cache in (one.expand(4, 128, 16), flat.as_strided((4, 128, 16), (64 * 16, 16, 1)), flat.as_strided((4, 128, 16), (127 * 16, 16, 1)),
                  flat.as_strided((4, 128, 16), (8, 64, 1)), flat[:16].expand(4, 128, 16)):
        with pytest.raises(ValueError):
            kvip_amd.PageTables(torch, **make, caches=[cache])
    # Places first, pages in between, one page, rows with room behind them: no row overlaps another.
    good = [flat[:128 * 4 * 16].view(128, 4, 16).transpose(0, 1), flat.view(4, 2, 128, 16)[:, 1], flat.as_strided((4, 128, 16), (128 * 20, 20, 1)),
            flat.as_strided((4, 128, 16), (127 * 20 + 16, 20, 1))]
    for cache in good:
        kvip_amd.PageTables(torch, **make, caches=[cache])
    kvip_amd.PageTables(torch, **{**make, "num_blocks": 1}, caches=[one])
    kvip_amd.PageTables(torch, **make, caches=[good[0][..., :8], good[0][..., 8:]])
    for twice in ([good[0], good[0]], [good[0], good[1], good[0][..., :4]]):
        with pytest.raises(ValueError):
            kvip_amd.PageTables(torch, **make, caches=twice)


def test_rows_move_in_a_cache_of_places_first(torch_gpu):
    torch = torch_gpu
    say("case places first")
    data = (torch.arange(128 * 4 * 16, device="cuda") % 251).to(torch.uint8).view(128, 4, 16)
    want = data.clone()
    op = kvip_amd.PageTables(torch, batch=1, max_context=512, num_blocks=4, max_tokens=16, device="cuda", caches=[data.transpose(0, 1)])
    op.extend(device(torch, [6], torch.int32))
    op.commit(device(torch, [3], torch.int32), device(torch, [[0, 2, 5]], torch.int32))
    want[1, 0], want[2, 0] = want[2, 0].clone(), want[5, 0].clone()
    assert torch.equal(data, want) and int(op.status.item()) == 0


# --- paths of many places ---------------------------------------------------------------------


def test_paths_longer_than_a_tree_move_every_row(torch_gpu):
    """A chain has no limit of 64 tokens, nor has the path that names those kept; a path that falls behind place 64
    stops there, and a count above the path's places is reported."""
    torch = torch_gpu
    say("case long paths")
    rng = np.random.default_rng(17)
    kept, steps, places = [150, 64, 65, 200, 129], [300, 200, 66, 201, 140], 150
    cache = torch.from_numpy(rng.integers(0, 256, (30, 128, 656))).to(torch.uint8).cuda()
    op = kvip_amd.PageTables(torch, batch=5, max_context=512, num_blocks=30, max_tokens=1000, device="cuda", caches=[cache])
    op.extend(device(torch, [100, 0, 127, 5, 90], torch.int32))
    op.commit(op.steps.clone())
    op.extend(device(torch, steps, torch.int32))
    path = np.full((5, places), -1, np.int32)
    for b in range(5):
        n = min(kept[b], places)
        path[b, :n] = np.sort(rng.choice(steps[b], n, replace=False))
    path[4, 100] = path[4, 99]  # does not rise
    table, bases = op.block_table.cpu().numpy().copy(), op.bases.tolist()
    rows = cache.cpu().numpy().copy().reshape(-1, 656)
    assert int(op.status.item()) == 0
    op.commit(device(torch, kept, torch.int32), device(torch, path, torch.int32))
    assert int(op.status.item()) == abi.STATUS_BAD_TREE | abi.STATUS_BAD_LENGTH
    assert op.lengths.tolist() == [n + k for n, k in zip(bases, kept)]
    want = rows.copy()
    for b, n in enumerate((150, 64, 65, 150, 100)):
        for i in range(n):
            src, dst = bases[b] + path[b, i], bases[b] + i
            want[table[b, dst // 128] * 128 + dst % 128] = rows[table[b, src // 128] * 128 + src % 128]
    assert np.array_equal(cache.cpu().numpy().reshape(want.shape), want)


# --- row counts that leave the arrays ---------------------------------------------------------


def test_rows_past_the_arrays_are_reported(torch_gpu):
    """cu_seqlens that go past the rows of the query or the probabilities, or fall: reported, and the requests that
    lie in the arrays as ever."""
    torch = torch_gpu
    say("case rows past the arrays")
    step = Step(torch, np.random.default_rng(3), [3, 4, 2], [100, 200, 50], 16)
    op = step.run(nodes=4)
    query, kv, table, lens, cu, visible = op._bound[:6]
    for ends in ([0, 3, 7, step.tokens + 1], [0, 3, 7, 6], [0, 3, 7, 1 << 30]):
        op.status.zero_()
        op.bind(query, kv, table, lens, device(torch, ends, torch.int32), visible)
        q, got = step.query.double().numpy(), host(op())
        for b in (0, 1):
            rows = step.rows[[step.slot(b, p) for p in range(step.lens[b])]]
            for i in range(step.counts[b]):
                at, sees = step.cu[b] + i, np.ones(step.lens[b], bool)
                sees[step.contexts[b]:] = [bool(int(step.bits[at]) >> j & 1) for j in range(step.counts[b])]
                want, _, bound, _ = draft.tree_attention(q[at], rows, sees, SCALE)
                assert np.all(np.abs(got[at] - want) <= bound + np.abs(want) * HALF_STEP["bf16"])
        assert int(op.status.item()) == abi.STATUS_BAD_LENGTH, ends
    case = verify_case(torch, np.random.default_rng(4), [3, 4, 2], 500, "chain", "fp32")
    for ends in ([0, 3, 7, 12], [0, 3, 7, 6], [0, 3, 7, 1 << 30]):
        op = run_verify(torch, {**case, "cu": np.asarray(ends)}, nodes=5, vocab=500)
        op()
        assert int(op.status.item()) & abi.STATUS_BAD_LENGTH, ends
        first = run_verify(torch, case, nodes=5, vocab=500)
        first()
        assert int(first.status.item()) == 0
        assert torch.equal(op.out_tokens[:2], first.out_tokens[:2]) and torch.equal(op.path[:2], first.path[:2])


# --- a scale of zero --------------------------------------------------------------------------


def test_a_zero_scale_weighs_all_rows_alike(torch_gpu):
    """Also where the products that it is applied to are 10^31."""
    say("case zero scale")
    step = Step(torch_gpu, np.random.default_rng(23), [3, 2], [260, 70], 16)
    scales = step.rows[:, 640:656].copy().view("<f4")
    step.rows[:, 640:656] = (scales * np.float32(1e30)).view(np.uint8)
    for scale in (0.0, -0.0):
        op = step.run(scale=scale)
        step.check(op, scale=scale)
        assert int(op.status.item()) == 0


# --- the tables' tensors in the framework's indexer -------------------------------------------


def test_the_indexer_selects_by_the_tables(torch_gpu):
    """A step of chains: kvip_amd.PrefillIndexer on the tables' cu_seqlens, lengths and block_table selects what it
    selects with the same made on the host, and a row sees the context and the step's rows up to its own."""
    torch = torch_gpu
    say("case indexer by the tables")
    rng = np.random.default_rng(29)
    before, counts = [700, 3000, 0, 130], [5, 12, 3, 1]
    op = kvip_amd.PageTables(torch, batch=4, max_context=4096, num_blocks=60, max_tokens=4000, device="cuda")
    model = draft.Tables(4, 32, 60, 4000)
    for step in (before, counts):
        op.extend(device(torch, step, torch.int32))
        model.extend(step)
        if step is before:
            op.commit(op.steps.clone())
            model.commit(before)
    rows = sum(counts)
    query = torch.randn((rows, 64, 128), device="cuda").to(torch.float8_e4m3fn)
    key = torch.randn((60, 128, 128), device="cuda").to(torch.float8_e4m3fn)
    weights = torch.randn((rows, 64), device="cuda")
    table = np.zeros((4, 32), np.int32)
    for b, pages in enumerate(model.pages):
        table[b, :len(pages)] = pages
    indexer = kvip_amd.PrefillIndexer(torch, max_rows=rows, max_context=4096, max_sequences=4, device="cuda")
    host_made = (device(torch, np.concatenate([[0], np.cumsum(counts)]), torch.int32), device(torch, model.lengths, torch.int32),
                 device(torch, table, torch.int32))
    want = indexer(query, weights, None, key, None, *host_made).clone()
    got = indexer(query, weights, None, key, None, op.cu_seqlens, op.lengths, op.block_table)
    assert torch.equal(got, want) and int(indexer.status.item()) == 0 and int(op.status.item()) == 0
    at = 0
    for b, n in enumerate(counts):
        for i in range(n):
            chosen = [x for x in got[at].tolist() if x >= 0]
            assert len(set(chosen)) == len(chosen) == min(before[b] + i + 1, 2048) and max(chosen) <= before[b] + i
            at += 1


# --- the most rows a request can have ---------------------------------------------------------


def test_all_heads_and_all_step_tokens(torch_gpu):
    say("case 128 heads of 64 tokens")
    step = Step(torch_gpu, np.random.default_rng(41), [64, 64, 1], [300, 10, 1000], 128)
    op = step.run()
    step.check(op)
    assert int(op.status.item()) == 0
