"""GPU tests of what the drafted round's operators promise at the edges of their rules: steps without
parents, requests that got no pages, targets whose support was drafted whole, workspaces of several
shapes, latents and scales at the ends of their range. Against oracle/draft.py, with the bounds of
tests/test_gpu_draft.py."""
import numpy as np
import pytest

import kvip_amd
from oracle import draft
from tests.test_gpu_draft import HALF_STEP, ROW, SCALE, Round, device, host, random_parents, same_tables, say

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
