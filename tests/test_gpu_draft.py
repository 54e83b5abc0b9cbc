"""GPU parity of the drafted round's operators (kvip_amd.PageTables, Rotary, KvRowStore, TreeAttention,
DraftVerifier) against oracle/draft.py, which works in 64 bits.

Whole numbers (pages, slots, positions, bits, tokens, stored codes and scales) have to be equal.
Tolerances: a rounding is off by at most half a step (bf16 2^-8, fp16 2^-11, fp32 2^-24 of the value). A
turned feature a cos - b sin has, besides its final rounding, an angle off by 2 pi 2^-25 (the fraction of a turn
in 32 bits) and sine and cosine off by 2 units of 2^-24 and three products and sums: 2^-20 (|a| + |b|) covers them.
Attention: the bounds that oracle/draft.py derives, and the output's rounding."""
import math

import numpy as np
import pytest

import kvip_amd
from kvip_amd.runtime import abi
from oracle import draft

pytestmark = pytest.mark.gpu
ROW = 656
SCALE = 576 ** -0.5
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def say(*args):
    print(*args, flush=True)


def dtype_of(torch, name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[name]


def host(x):
    return x.double().cpu().numpy() if x.is_floating_point() else x.cpu().numpy()


def device(torch, values, dtype):
    return torch.from_numpy(np.ascontiguousarray(values)).to(dtype).cuda()


# --- rotary ---------------------------------------------------------------------------------


def turn_bound(x, frequencies, half, magnitude, want, step):
    pairs = len(frequencies)
    first, second = (slice(0, pairs), slice(pairs, 2 * pairs)) if half else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
    sums = np.zeros_like(want)
    sums[..., first] = sums[..., second] = (np.abs(x[..., first]) + np.abs(x[..., second])) * magnitude
    return sums * 2.0 ** -20 + np.abs(want) * step


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("tokens,heads,rotary,dim,skip", [(1, 1, 64, 64, 0), (5, 3, 6, 7, 1), (33, 16, 64, 128, 64),
                                                            (7, 128, 64, 64, 512), (300, 1, 32, 33, 3), (2, 5, 512, 512, 0),
                                                            (1500, 2, 16, 24, 8)])
def test_rotary_matches(torch_gpu, dtype, half, tokens, heads, rotary, dim, skip):
    torch = torch_gpu
    rng = np.random.default_rng(tokens * heads + rotary)
    say(f"case rotary {dtype} half={half} tokens={tokens} heads={heads} rotary={rotary} dim={dim} skip={skip}")
    t = dtype_of(torch, dtype)
    scaling = {"kind": "yarn", "factor": 8.0, "original": 4096} if heads == 16 else None
    op = kvip_amd.Rotary(torch, rotary_dim=rotary, layout="half" if half else "interleaved", scaling=scaling, device="cuda")
    frequencies = op.frequencies.cpu().numpy()
    positions = rng.integers(0, 1 << 20, tokens)
    positions[0] = -3 if tokens > 1 else 1 << 20
    whole = device(torch, rng.standard_normal((tokens, heads, skip + dim)), t)
    keys = device(torch, rng.standard_normal((tokens, dim)), t)
    x, k = host(whole[..., skip:]), host(keys)
    out = torch.full((heads, tokens, dim + 1), 7.0, dtype=t, device="cuda")  # heads first, rows one apart
    y = out.transpose(0, 1)[..., :dim]
    op.bind(device(torch, positions, torch.int64), whole[..., skip:], keys, query_out=y)
    got, key = op()
    assert got is y and key is keys
    for have, from_, what in ((y, x, "query"), (keys, k, "key")):  # into another array, and in place
        want = draft.turned(from_, positions, frequencies, half, op.magnitude)
        bound = turn_bound(from_, frequencies, half, op.magnitude, want, HALF_STEP[dtype])
        off = np.abs(host(have) - want)
        assert np.all(off <= bound), (what, float(off.max()))
        assert np.array_equal(host(have)[..., rotary:], from_[..., rotary:])
    assert torch.all(out[..., dim:] == 7.0) and np.array_equal(host(whole[..., skip:]), x)


def test_rotary_and_store_of_more_tokens_than_a_launch(torch_gpu):
    torch = torch_gpu
    say("case rotary and store of 2^22 + 5 tokens")
    n = (1 << 22) + 5
    rotary = kvip_amd.Rotary(torch, rotary_dim=2, device="cuda")
    x = torch.randn((1, 2), device="cuda").repeat(n, 1)
    positions = torch.arange(n, device="cuda") % 1000
    rotary.bind(positions, x)()
    assert torch.equal(x[1000:], x[:n - 1000]) and not torch.equal(x[0], x[1])
    kv = torch.zeros((2, 128, ROW), dtype=torch.uint8, device="cuda")
    latent = torch.randn((1, 576), device="cuda").to(torch.bfloat16).expand(n, 576)
    slots = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    slots[0], slots[-1] = 7, 200
    kvip_amd.KvRowStore(torch, kv_cache=kv).bind(latent[:, :512], latent[:, 512:], slots)()
    flat = kv.view(256, ROW)
    assert bool(flat[7].any()) and torch.equal(flat[7], flat[200]) and int(flat.any(1).sum()) == 2


def test_rotary_inverse_is_the_gradient(torch_gpu):
    """<turn(x), g> = <x, back(g)> for the turn's gradient, and differences of the turned features."""
    torch = torch_gpu
    say("case rotary inverse")
    gen = torch.Generator(device="cuda").manual_seed(1)
    positions = torch.randint(0, 5000, (40,), generator=gen, device="cuda")
    x, g = (torch.randn((40, 4, 64), generator=gen, device="cuda") for _ in range(2))
    for layout in ("interleaved", "half"):
        op = kvip_amd.Rotary(torch, rotary_dim=64, layout=layout, device="cuda")
        y, back = torch.empty_like(x), torch.empty_like(x)
        op.bind(positions, x, query_out=y)()
        op.bind(positions, g, query_out=back, inverse=True)()
        left, right = (y.double() * g.double()).sum(), (x.double() * back.double()).sum()
        size = float((x.double().abs() * back.double().abs()).sum())
        assert abs(float(left - right)) <= 2 * 2.0 ** -20 * 2 * size
        step = torch.randn((40, 4, 64), generator=gen, device="cuda")
        moved = torch.empty_like(x)
        op.bind(positions, x + 0.5 * step, query_out=moved)()
        difference = ((moved.double() - y.double()) / 0.5 * g.double()).sum()
        slope = (step.double() * back.double()).sum()
        assert abs(float(difference - slope)) <= 2.0 ** -16 * float((step.abs() * back.abs()).double().sum() + size)
        op.bind(positions, y, inverse=True)()  # in place, and back to where it was
        assert float((y - x).abs().max()) <= 2.0 ** -18 * float(x.abs().max()) * 2


def test_rotary_refuses(torch_gpu):
    torch = torch_gpu
    op = kvip_amd.Rotary(torch, rotary_dim=8, device="cuda")
    positions = torch.zeros(4, dtype=torch.int64, device="cuda")
    x = torch.zeros((4, 2, 8), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        op()
    for query, kw in ((x[:3], {}), (x[..., :6], {}), (x.double(), {}), (x.cpu(), {}), (x.transpose(1, 2), {}),
                      (x, dict(key=x.float())), (x, dict(key_out=x)), (x, dict(query_out=x.float())),
                      (x, dict(query_out=x[:, :1].expand(4, 2, 8))), (x, dict(query_out=x.view(-1).as_strided((4, 2, 8), (8, 8, 1)))),
                      (x[:, :1].expand(4, 2, 8), {})):
        with pytest.raises(ValueError):
            op.bind(positions, query, **kw)
    for bad in (positions.int(), positions.cpu(), positions.view(2, 2), torch.zeros(8, dtype=torch.int64, device="cuda")[::2]):
        with pytest.raises(ValueError):
            op.bind(bad, x)
    empty = op.bind(positions[:0], x[:0])()
    assert empty[0].shape[0] == 0


# --- rows ------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,layout,stride", [(1, "interleaved", 656), (5, None, 672), (131, "half", 656)])
def test_stored_rows_match(torch_gpu, dtype, tokens, layout, stride):
    torch = torch_gpu
    rng = np.random.default_rng(tokens)
    say(f"case store {dtype} tokens={tokens} layout={layout} stride={stride}")
    t = dtype_of(torch, dtype)
    kv = device(torch, rng.integers(0, 256, (4, 128, stride)), torch.uint8)
    before = kv.cpu().numpy().reshape(-1, stride)
    projected = rng.standard_normal((tokens, 577)) * np.exp(rng.uniform(-4, 4, (tokens, 1)))
    projected[0, 128:256] = 0
    projected[tokens // 2, :128] *= 1e-30  # bf16 and fp32: tiny scales; fp16: zeros
    projected[tokens // 2, 3] = 5e-40      # below the normal range
    x = device(torch, projected, t)
    slots = rng.permutation(512)[:tokens].astype(np.int64)
    if tokens > 1:
        slots[1], slots[2] = -1, 512  # a padded token, and one past the cache
    rotary = None if layout is None else kvip_amd.Rotary(torch, rotary_dim=64, layout=layout, device="cuda")
    positions = rng.integers(0, 100000, tokens)
    op = kvip_amd.KvRowStore(torch, kv_cache=kv, rotary=rotary)
    out = op.bind(x[:, :512], x[:, 512:576], device(torch, slots, torch.int64),
                  None if rotary is None else device(torch, positions, torch.int64))()
    got = out.cpu().numpy().reshape(-1, stride)
    assert int(op.status.item()) == (abi.STATUS_BAD_TOKEN if tokens > 1 else 0)
    values = host(x)
    codes, scales = draft.stored_rows(values[:, :512])
    rope, bound = values[:, 512:576], np.abs(values[:, 512:576]) * 2.0 ** -8
    if rotary is not None:
        f = rotary.frequencies.cpu().numpy()
        want = draft.turned(rope, positions, f, layout == "half")
        rope, bound = want, turn_bound(rope, f, layout == "half", 1.0, want, 2.0 ** -8)
    kept = [i for i in range(tokens) if 0 <= slots[i] < 512]
    for i in kept:
        row = got[slots[i]]
        assert np.array_equal(row[640:656].view("<f4"), scales[i])
        assert np.array_equal(row[:512], codes[i]), i
        have = (row[512:640].view("<u2").astype(np.uint32) << 16).view(np.float32)
        assert np.all(np.abs(have - rope[i]) <= bound[i])
        assert np.array_equal(row[656:], before[slots[i]][656:])
    others = np.setdiff1d(np.arange(512), slots[kept])
    assert np.array_equal(got[others], before[others])


def test_row_store_refuses(torch_gpu):
    torch = torch_gpu
    kv = torch.zeros((2, 128, 656), dtype=torch.uint8, device="cuda")
    x = torch.zeros((4, 576), dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    op = kvip_amd.KvRowStore(torch, kv_cache=kv)
    with pytest.raises(ValueError):
        op()
    for latent, rope, at, positions in ((x[:, :500], x[:, 512:], slots, None), (x[:, :512], x[:, 500:], slots, None),
                                        (x[:, :512], x[:, 512:].float(), slots, None), (x[:, :512], x[:, 512:], slots.int(), None),
                                        (x[:, :512], x[:, 512:], slots[:3], None), (x[:, :512], x[:, 512:], slots, slots),
                                        (x[:, :512].cpu(), x[:, 512:], slots, None)):
        with pytest.raises(ValueError):
            op.bind(latent, rope, at, positions)
    turned = kvip_amd.KvRowStore(torch, kv_cache=kv, rotary=kvip_amd.Rotary(torch, rotary_dim=64, device="cuda"))
    with pytest.raises(ValueError):
        turned.bind(x[:, :512], x[:, 512:], slots)
    for bad in (kv.float(), kv[:, :64], kv[..., :640], kv.transpose(1, 2)):
        with pytest.raises(ValueError):
            kvip_amd.KvRowStore(torch, kv_cache=bad)
    with pytest.raises(ValueError):
        kvip_amd.KvRowStore(torch, kv_cache=kv, rotary=kvip_amd.Rotary(torch, rotary_dim=32, device="cuda"))
    with pytest.raises(ValueError):  # 16-byte steps
        kvip_amd.KvRowStore(torch, kv_cache=torch.zeros((2, 128, 660), dtype=torch.uint8, device="cuda")).bind(
            x[:, :512], x[:, 512:], slots)()
    assert op.bind(x[:0, :512], x[:0, 512:], slots[:0])() is not None


# --- page tables -----------------------------------------------------------------------------


def same_tables(op, model):
    table = np.full((op.batch, op.max_blocks), -1)
    for b, pages in enumerate(model.pages):
        table[b, :len(pages)] = pages
    assert np.array_equal(op.block_table.cpu().numpy(), table)
    assert op.lengths.tolist() == model.lengths and op.bases.tolist() == model.bases and op.steps.tolist() == model.steps
    count = int(op.free_count.item())
    assert op.free.tolist()[:count] == model.stack
    assert int(op.ticket.item()) == 0


def random_parents(rng, counts, total):
    parents, at = np.full(total, -1, np.int32), 0
    for n in counts:
        for i in range(1, min(n, total - at)):
            parents[at + i] = rng.integers(-1 if rng.random() < 0.1 else 0, i)
        at += max(n, 0)
    return parents


@pytest.mark.parametrize("batch,blocks,pages,rows,trees", [(1, 1, 1, 1, False), (3, 5, 9, 40, True), (70, 9, 200, 900, True),
                                                           (257, 33, 3000, 20000, False), (1024, 4, 1500, 4096, True)])
def test_tables_follow_the_model(torch_gpu, batch, blocks, pages, rows, trees):
    torch = torch_gpu
    rng = np.random.default_rng(batch)
    say(f"case tables batch={batch} blocks={blocks} pages={pages} rows={rows} trees={trees}")
    op = kvip_amd.PageTables(torch, batch=batch, max_context=blocks * 128, num_blocks=pages, max_tokens=rows, device="cuda")
    model = draft.Tables(batch, blocks, pages, rows)
    same_tables(op, model)
    for step in range(8):
        most = 65 if trees and step != 5 else 66 if trees else 300
        counts = rng.integers(-1 if step == 3 else 0, min(most, 2 + 2 * rows // batch), batch)
        counts[rng.random(batch) < 0.2] = 0
        if step == 6:
            counts[rng.integers(0, batch)] = (1 << 31) - 1
        parents = None
        if trees and step % 3 != 2:
            parents = random_parents(rng, counts, rows)
            if step == 4:
                parents[rng.integers(0, rows)] = 63
        op.status.zero_()
        cu, slots, positions = op.extend(device(torch, counts, torch.int32),
                                         None if parents is None else device(torch, parents, torch.int32))
        want = model.extend(counts.tolist(), parents)
        assert cu.tolist() == want[0], step
        assert slots.tolist() == want[1] and positions.tolist() == want[2], step
        if parents is not None:
            assert [x & (1 << 64) - 1 for x in op.visible.tolist()] == want[3], step
        assert int(op.status.item()) == want[4], (step, want[4])
        same_tables(op, model)
        if step % 2:
            lengths = rng.integers(0, blocks * 128, batch)
            lengths = np.minimum(lengths, model.lengths) if step == 1 else lengths
            op.truncate(device(torch, lengths, torch.int32))
            model.truncate(lengths.tolist())
        else:
            kept = rng.integers(0, 66, batch)
            op.commit(device(torch, kept, torch.int32))
            model.commit(kept.tolist())
        same_tables(op, model)


def test_a_truncate_undoes_an_extend(torch_gpu):
    torch = torch_gpu
    say("case tables undone")
    op = kvip_amd.PageTables(torch, batch=5, max_context=2048, num_blocks=60, max_tokens=2000, device="cuda")
    op.extend(device(torch, [100, 128, 0, 129, 400], torch.int32))
    before = [t.clone() for t in (op.block_table, op.lengths, op.free, op.free_count)]
    lengths = op.lengths.clone()
    op.extend(device(torch, [29, 300, 1, 0, 700], torch.int32))
    assert int(op.free_count.item()) < int(before[3].item())
    op.truncate(lengths)
    assert all(torch.equal(a, b) for a, b in zip(before, (op.block_table, op.lengths, op.free, op.free_count)))
    assert int(op.status.item()) == 0


def test_kept_rows_move_together(torch_gpu):
    """Rows of three caches (KV rows, index keys, scales) and a padded one; a path that falls, and one
    past the step, stop at the bad entry."""
    torch = torch_gpu
    rng = np.random.default_rng(8)
    say("case tables move")
    pages = 12
    caches = [device(torch, rng.integers(0, 256, (pages, 128, 656)), torch.uint8),
              device(torch, rng.integers(0, 256, (pages + 2, 128, 128)), torch.uint8),
              torch.randn((pages, 128), device="cuda"),
              device(torch, rng.integers(0, 256, (pages, 128, 1, 672)), torch.uint8)[..., :656]]
    op = kvip_amd.PageTables(torch, batch=5, max_context=512, num_blocks=pages, max_tokens=200, device="cuda", caches=caches)
    op.extend(device(torch, [125, 0, 1, 7, 10], torch.int32))
    op.commit(op.steps.clone())
    op.extend(device(torch, [20, 3, 40, 6, 4], torch.int32), torch.full((200,), -1, dtype=torch.int32, device="cuda"))
    path = np.full((5, 30), -1, np.int32)
    kept = np.asarray([5, 0, 30, 3, 3])
    path[0, :5], path[2, :30], path[3, :3], path[4, :3] = [0, 2, 3, 9, 19], np.arange(30) + 10, [0, 4, 2], [0, 1, 4]
    table, bases = op.block_table.cpu().numpy().copy(), op.bases.tolist()
    before = [c.cpu().numpy().copy().reshape(c.shape[0] * 128, -1) for c in caches]
    op.commit(device(torch, kept, torch.int32), device(torch, path, torch.int32))
    assert int(op.status.item()) == abi.STATUS_BAD_TREE
    assert op.lengths.tolist() == [130, 0, 31, 10, 13]
    for cache, rows in zip(caches, before):
        want = rows.copy()
        for b, good in ((0, 5), (2, 30), (3, 2), (4, 2)):
            for i in range(good):
                src, dst = bases[b] + path[b, i], bases[b] + i
                want[table[b, dst // 128] * 128 + dst % 128] = rows[table[b, src // 128] * 128 + src % 128]
        assert np.array_equal(cache.cpu().numpy().reshape(want.shape), want)


def test_page_tables_refuse(torch_gpu):
    torch = torch_gpu
    make = dict(batch=2, max_context=512, num_blocks=4, max_tokens=16, device="cuda")
    for cache in (torch.zeros((4, 128, 656), dtype=torch.uint8), torch.zeros((3, 128, 656), dtype=torch.uint8, device="cuda"),
                  torch.zeros((4, 64, 656), dtype=torch.uint8, device="cuda"), torch.zeros((4, 128, 2), dtype=torch.uint8, device="cuda"),
                  torch.zeros((4, 128, 8, 8), device="cuda").transpose(2, 3)):
        with pytest.raises(ValueError):
            kvip_amd.PageTables(torch, **make, caches=[cache])
    op = kvip_amd.PageTables(torch, **make)
    two = torch.zeros(2, dtype=torch.int32, device="cuda")
    for counts, parents in ((two.long(), None), (two[:1], None), (two.cpu(), None), (two, two), (two, torch.zeros(16, device="cuda"))):
        with pytest.raises(ValueError):
            op.extend(counts, parents)
    for kept, path in ((two.float(), None), (two, two), (two, torch.zeros((3, 4), dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            op.commit(kept, path)
    with pytest.raises(ValueError):
        op.truncate(two.long())


# --- attention -------------------------------------------------------------------------------


class Step:
    """A packed step over a shuffled cache: counts[b] step tokens, contexts[b] rows before them."""

    def __init__(self, torch, rng, counts, contexts, heads, *, stride=656, tree=True, spare=3, pad=2):
        self.torch, self.counts, self.contexts, self.heads = torch, counts, contexts, heads
        lens = [c + n for c, n in zip(contexts, counts)]
        blocks = [-(-x // 128) for x in lens]
        self.pages = sum(blocks) + spare
        width = max(max(blocks), 1)
        order, at = rng.permutation(self.pages), 0
        self.table = np.full((len(counts), width), -7, np.int32)  # entries past a request's pages are not read
        for b, n in enumerate(blocks):
            self.table[b, :n] = order[at:at + n]
            at += n
        rows = np.zeros((self.pages * 128, stride), np.uint8)
        rows[:, :512] = draft.e4m3_bytes(np.clip(rng.standard_normal((len(rows), 512)) * 120, -448, 448).astype(np.float32))
        rope = rng.standard_normal((len(rows), 64)).astype(np.float32)
        rows[:, 512:640] = (rope.view(np.uint32) >> 16).astype("<u2").view(np.uint8)
        rows[:, 640:656] = (rng.uniform(0.2, 1.5, (len(rows), 4)) / 120).astype("<f4").view(np.uint8)
        rows[:, 656:] = 0xFF
        self.rows, self.lens = rows, lens
        self.tokens = sum(counts) + pad
        self.cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.bits = np.zeros(self.tokens, np.uint64)
        for b, n in enumerate(counts):
            parents = [-1] + [int(rng.integers(-1 if tree and rng.random() < 0.1 else 0, i)) if tree else i - 1 for i in range(1, n)]
            self.bits[self.cu[b]:self.cu[b] + n] = np.asarray(draft.ancestors(parents[:n])[0], np.uint64) if n else []
        self.query = torch.from_numpy(rng.standard_normal((self.tokens, heads, 576)).astype(np.float32)).to(torch.bfloat16)

    def slot(self, b, position):
        return self.table[b, position // 128] * 128 + position % 128

    def run(self, *, nodes=None, output="bf16", scale=SCALE, visible=True, lse=True):
        torch = self.torch
        kv = torch.from_numpy(self.rows).cuda().view(self.pages, 128, -1)
        op = kvip_amd.TreeAttention(torch, batch=len(self.counts), heads=self.heads, max_nodes=nodes or max(max(self.counts), 1),
                                    max_tokens=self.tokens, max_context=self.table.shape[1] * 128, device="cuda",
                                    output_dtype=dtype_of(torch, output), lse=lse)
        op.output.fill_(3.0)
        if lse:
            op.lse.fill_(3.0)
        op.bind(self.query.cuda(), kv, device(torch, self.table, torch.int32), device(torch, self.lens, torch.int32),
                device(torch, self.cu, torch.int32), device(torch, self.bits.view(np.int64), torch.int64) if visible else None,
                scale)
        return op

    def check(self, op, *, output="bf16", scale=SCALE, only=None):
        got = host(op())
        lse = None if op.lse is None else host(op.lse)
        worst, q = 0.0, self.query.double().numpy()
        for b, n in enumerate(self.counts):
            if only is not None and b not in only:
                continue
            rows = self.rows[[self.slot(b, p) for p in range(self.lens[b])]]
            for i in range(n):
                row = self.cu[b] + i
                sees = np.ones(self.lens[b], bool)
                sees[self.lens[b] - n:] = [bool(int(self.bits[row]) >> j & 1) for j in range(n)]
                want, want_lse, bound, lse_bound = draft.tree_attention(q[row], rows, sees, scale)
                bound = bound + np.abs(want) * HALF_STEP[output]
                off = np.abs(got[row] - want)
                assert np.all(off <= bound), (b, i, float((off - bound).max()))
                worst = max(worst, float((off / np.maximum(bound, 1e-30)).max()))
                if lse is not None:
                    assert np.all((lse[row] == want_lse) | (np.abs(lse[row] - want_lse) <= lse_bound)), (b, i)
        say(f"  largest share of the bound {worst:.2f}")
        behind = self.cu[-1]
        assert np.all(got[behind:] == 3.0) and (lse is None or np.all(lse[behind:] == 3.0))


@pytest.mark.parametrize("heads,counts,contexts", [
    (16, [1], [0]), (1, [1], [1]), (16, [2], [31]), (5, [3, 0, 1], [62, 0, 100]), (16, [4, 4], [128, 700]),
    (16, [3, 4, 1], [1000, 0, 95]), (20, [3, 1, 2], [129, 31, 33]), (128, [1, 2], [300, 127]), (32, [7, 5, 9], [511, 1, 2000]),
    (8, [64, 13], [40, 4000]), (128, [3], [1500]), (16, [1] * 40, list(range(7, 207, 5))), (33, [2, 1], [900, 40]),
    (16, [4] * 70, [(37 * i) % 600 for i in range(70)])])
def test_tree_attention_matches(torch_gpu, heads, counts, contexts):
    say(f"case tree heads={heads} counts={counts[:6]} contexts={contexts[:6]}")
    step = Step(torch_gpu, np.random.default_rng(heads + len(counts)), counts, contexts, heads)
    op = step.run()
    step.check(op)
    assert int(op.status.item()) == 0


@pytest.mark.parametrize("heads,requests,longest", [(2, 400, 5000), (96, 48, 8000), (40, 30, 9000), (2, 700, 900), (3, 1024, 400),
                                                   (40, 2, 30000)])
def test_tree_attention_many_long_requests(torch_gpu, heads, requests, longest):
    """More steps than workgroups take at a time, of requests with shared pages and of some without tokens:
    shares that start, end and pass through several requests."""
    torch = torch_gpu
    say(f"case tree many heads={heads} requests={requests} longest={longest}")
    rng = np.random.default_rng(heads)
    step = Step(torch, rng, [1], [127], heads, spare=149, pad=requests + 4)
    counts = [int(rng.random() < 0.9) * (1 + int(heads == 40 and rng.random() < 0.7)) for _ in range(requests)]
    lens = [int(rng.integers(n, longest)) if rng.random() < 0.8 else n for n in counts]
    step.counts, step.lens, step.contexts = counts, lens, [x - n for x, n in zip(lens, counts)]
    step.table = rng.integers(0, step.pages, (requests, -(-longest // 128))).astype(np.int32)
    step.cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    step.tokens = int(step.cu[-1]) + 2
    step.query = torch.from_numpy(rng.standard_normal((step.tokens, heads, 576)).astype(np.float32)).to(torch.bfloat16)
    step.bits = np.zeros(step.tokens, np.uint64)
    for b, n in enumerate(counts):
        step.bits[step.cu[b]:step.cu[b] + n] = [(1 << (i + 1)) - 1 for i in range(n)]
    op = step.run()
    step.check(op)
    assert int(op.status.item()) == 0
    first = op.output.clone()
    assert torch.equal(op(), first)  # joined in one order


def test_tree_attention_options(torch_gpu):
    """fp32 output without log-sum-exp, padded rows, another scale, more max_nodes than any request has, a
    chain without bits, and the functional form."""
    torch = torch_gpu
    say("case tree options")
    step = Step(torch, np.random.default_rng(5), [3, 2], [260, 700], 12, stride=720, tree=False)
    op = step.run(nodes=11, output="fp32", scale=0.11, visible=False, lse=False)
    step.check(op, output="fp32", scale=0.11)
    kv = torch.from_numpy(step.rows).cuda().view(step.pages, 128, 1, 720)
    again = kvip_amd.tree_attention(step.query.cuda(), kv, device(torch, step.table, torch.int32),
                                    device(torch, step.lens, torch.int32), device(torch, step.cu, torch.int32), scale=0.11,
                                    output_dtype=torch.float32, max_nodes=11)
    assert torch.equal(again[:5], op.output[:5])
    negative = step.run(scale=-0.05)
    step.check(negative, scale=-0.05)
    zero = step.run(scale=0.0)
    step.check(zero, scale=0.0)


def test_tree_attention_rows_that_see_nothing(torch_gpu):
    say("case tree empty rows")
    step = Step(torch_gpu, np.random.default_rng(6), [4, 3], [0, 40], 16)
    step.bits[1] = 0         # sees nothing at all
    step.bits[2] = 1 << 3    # only the last token
    step.bits[5] = 0         # its context alone
    op = step.run()
    step.check(op)
    assert not op.output[1].any() and bool((op.lse[1] == -math.inf).all())


@pytest.mark.parametrize("heads", [4, 12, 40])
def test_tree_attention_hidden_rows_hold_anything(torch_gpu, heads):
    """NaN features, scales and rotary features, and infinite scales, in step rows that a token does not see, behind
    the last row and in other pages do not reach it; rows that see one are NaN."""
    say(f"case tree hidden heads={heads}")
    step = Step(torch_gpu, np.random.default_rng(heads), [6, 5], [125, 700], heads)
    everyone = (1 << 6) - 1
    for b, n in enumerate(step.counts):
        for i in range(n):
            step.bits[step.cu[b] + i] = everyone & ~(1 << 1 | 1 << 3 | 1 << 4)
    step.bits[4] = 1 << 3                     # sees a NaN feature
    step.bits[step.cu[1] + 2] = 1 << 1        # sees an infinite scale
    rows, poison = step.rows, []
    for b in range(2):
        past = step.contexts[b]
        at = [step.slot(b, past + j) for j in (1, 3, 4)]
        rows[at[0], 640:656] = np.asarray([np.inf, 1, np.nan, 2], "<f4").view(np.uint8)
        rows[at[1], 5:9] = [0x7F, 0xFF, 0x7F, 0x30]
        rows[at[2], 512:640] = 0xFF
        poison += at
    used = {step.slot(b, p) for b in range(2) for p in range(step.lens[b])}
    rest = [r for r in range(len(rows)) if r not in used]
    rows[rest] = 0xFF
    want = Step.__new__(Step)
    want.__dict__.update(step.__dict__)
    want.rows = rows.copy()
    want.rows[poison, :512], want.rows[poison, 512:] = 0x38, 0  # hidden: any finite row does
    op = step.run()
    got = host(op())
    for row in (4, step.cu[1] + 2):
        assert np.all(np.isnan(got[row])) and bool(op.lse[row].isnan().all())
    q = step.query.double().numpy()
    for b, n in enumerate(step.counts):
        held = want.rows[[step.slot(b, p) for p in range(step.lens[b])]]
        for i in range(n):
            row = step.cu[b] + i
            if row in (4, step.cu[1] + 2):
                continue
            sees = np.ones(step.lens[b], bool)
            sees[step.lens[b] - n:] = [bool(int(step.bits[row]) >> j & 1) for j in range(n)]
            expected, _, bound, _ = draft.tree_attention(q[row], held, sees, SCALE)
            assert np.all(np.abs(got[row] - expected) <= bound + np.abs(expected) * 2.0 ** -8), (b, i)
    assert int(op.status.item()) == 0


def test_tree_attention_bad_tables_and_lengths(torch_gpu):
    torch = torch_gpu
    say("case tree bad tables")
    step = Step(torch, np.random.default_rng(9), [2, 2, 3], [500, 300, 200], 16)
    step.table[0, 1], step.table[0, 2] = step.pages, -1  # two of four pages are not there
    op = step.run()
    step.check(op, only=(1, 2))
    assert int(op.status.item()) == abi.STATUS_BAD_BLOCK
    q, got = step.query.double().numpy(), host(op.output)
    there = np.asarray([p // 128 not in (1, 2) for p in range(502)])
    rows = step.rows[[step.slot(0, p) if ok else 0 for p, ok in enumerate(there)]]
    for i in range(2):
        sees = there.copy()
        sees[500:] &= [bool(int(step.bits[i]) >> j & 1) for j in range(2)]
        want, _, bound, _ = draft.tree_attention(q[i], rows, sees, SCALE)
        assert np.all(np.abs(got[i] - want) <= bound + np.abs(want) * 2.0 ** -8)
    # Lengths past the table, below the step's tokens and below zero; more step tokens than max_nodes.
    step = Step(torch, np.random.default_rng(10), [2, 2, 3, 2], [500, 0, 100, 60], 16)
    step.lens[0], step.lens[1], step.lens[2] = 10 ** 6, 1, -5
    step.table[:] = np.maximum(step.table, 0)
    op = step.run(nodes=2)
    step.check(op, only=(3,))
    assert int(op.status.item()) == abi.STATUS_BAD_LENGTH
    assert not op.output[4:6].any() and bool((op.output[6] == 3.0).all())


def test_tree_attention_long_cache(torch_gpu):
    """Rows past the 4 GB of a cache, and a context long enough to be shared by many workgroups."""
    torch = torch_gpu
    say("case tree long cache")
    rng = np.random.default_rng(11)
    step = Step(torch, rng, [3], [20000], 16)
    blocks, first = 60000, 60000 - step.pages  # 5.04 GB
    kv = torch.zeros((blocks, 128, ROW), dtype=torch.uint8, device="cuda")
    kv[first:] = torch.from_numpy(step.rows).cuda().view(-1, 128, ROW)
    op = step.run()
    op.bind(step.query.cuda(), kv, device(torch, step.table + first, torch.int32), device(torch, step.lens, torch.int32),
            device(torch, step.cu, torch.int32), device(torch, step.bits.view(np.int64), torch.int64))
    step.check(op)
    # The stores reach there as well.
    x = torch.randn((2, 576), device="cuda").to(torch.bfloat16)
    slots = torch.tensor([blocks * 128 - 1, 3], device="cuda")
    kvip_amd.KvRowStore(torch, kv_cache=kv).bind(x[:, :512], x[:, 512:], slots)()
    codes, _ = draft.stored_rows(host(x)[:, :512])
    assert np.array_equal(kv[-1, -1, :512].cpu().numpy(), codes[0]) and np.array_equal(kv[0, 3, :512].cpu().numpy(), codes[1])


def test_tree_attention_refuses(torch_gpu):
    torch = torch_gpu
    op = kvip_amd.TreeAttention(torch, batch=2, heads=4, max_nodes=3, max_tokens=6, max_context=256, device="cuda")
    good = dict(query=torch.zeros((6, 4, 576), dtype=torch.bfloat16, device="cuda"),
                kv_cache=torch.zeros((4, 128, 656), dtype=torch.uint8, device="cuda"),
                block_table=torch.zeros((2, 2), dtype=torch.int32, device="cuda"),
                seq_lens=torch.zeros(2, dtype=torch.int32, device="cuda"),
                cu_seqlens=torch.zeros(3, dtype=torch.int32, device="cuda"),
                visible=torch.zeros(6, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        op()
    bad = dict(query=[good["query"].float(), good["query"][:5], good["query"].cpu(), good["query"].transpose(0, 1)],
               kv_cache=[good["kv_cache"].int(), good["kv_cache"][:, :64], good["kv_cache"][..., :640], good["kv_cache"].cpu()],
               block_table=[good["block_table"].long(), good["block_table"][:1], torch.zeros((2, 3), dtype=torch.int32, device="cuda"),
                            good["block_table"][:, :0]],
               seq_lens=[good["seq_lens"].long(), good["cu_seqlens"]], cu_seqlens=[good["seq_lens"], good["cu_seqlens"].long()],
               visible=[good["visible"].int(), good["visible"][:5]])
    for name, values in bad.items():
        for value in values:
            with pytest.raises(ValueError):
                op.bind(**{**good, name: value})
    for scale in (float("inf"), float("nan")):
        with pytest.raises(ValueError):
            op.bind(**good, scale=scale)
    with pytest.raises(ValueError):  # more steps than 32 bits count
        kvip_amd.TreeAttention(torch, batch=1024, heads=128, max_nodes=64, max_tokens=1, max_context=1 << 24, device="cuda")
    assert not op.bind(**good)().any()  # a step without tokens


# --- verification ----------------------------------------------------------------------------


def softmax_rows(rng, n, vocab, sharp=4.0):
    x = np.exp(sharp * rng.standard_normal((n, vocab)))
    return x / x.sum(1, keepdims=True)


def verify_case(torch, rng, counts, vocab, drafted, dtype, *, pad=2, width=0):
    total = sum(counts) + pad
    t = dtype_of(torch, dtype)
    wide = torch.zeros((total, vocab + width), dtype=t, device="cuda")
    probs = wide[:, :vocab]
    p = softmax_rows(rng, total, vocab)
    probs.copy_(torch.from_numpy(p))
    parents = draft_probs = None
    tokens = rng.integers(0, vocab, total)
    at = 0
    if drafted == "tree":
        parents = np.full(total, -1, np.int32)
    if drafted == "draft":
        q = 0.6 * p + 0.4 * softmax_rows(rng, total, vocab)
        draft_probs = device(torch, q, t)
    for n in counts:
        for i in range(1, n):
            up = int(rng.integers(max(0, i - 4), i)) if drafted == "tree" else i - 1
            if drafted == "tree":
                parents[at + i] = up
            source = q[at + up] if drafted == "draft" else p[at + up]
            tokens[at + i] = rng.choice(vocab, p=source / source.sum())
        at += n
    return dict(probs=probs, tokens=tokens, parents=parents, draft=draft_probs, cu=np.concatenate([[0], np.cumsum(counts)]),
                uniforms=rng.random(total).astype(np.float32), final=rng.random(len(counts)).astype(np.float32))


def run_verify(torch, case, *, nodes, vocab):
    op = kvip_amd.DraftVerifier(torch, batch=len(case["final"]), max_nodes=nodes, vocab=vocab, device="cuda")
    op.bind(case["probs"], device(torch, case["tokens"], torch.int64), device(torch, case["cu"], torch.int32),
            device(torch, case["uniforms"], torch.float32), device(torch, case["final"], torch.float32),
            parents=None if case["parents"] is None else device(torch, case["parents"], torch.int32), draft_probs=case["draft"])
    return op


def check_verify(case, op, *, nodes, limit=64):
    tokens, kept, path = (x.cpu().numpy() for x in op())
    probs = host(case["probs"].float())
    q = None if case["draft"] is None else host(case["draft"].float())
    for b in range(len(kept)):
        s = slice(case["cu"][b], min(case["cu"][b + 1], case["cu"][b] + limit))
        if s.start == s.stop:
            assert kept[b] == 0 and np.all(path[b] == -1) and np.all(tokens[b] == -1)
            continue
        want, out = draft.verify(probs[s], case["tokens"][s], None if case["parents"] is None else case["parents"][s],
                                 None if q is None else q[s], case["uniforms"][s], case["final"][b])
        assert kept[b] == len(want) and path[b].tolist() == want + [-1] * (nodes - len(want)), b
        assert tokens[b].tolist() == out + [-1] * (nodes - len(out)), b
    return kept


@pytest.mark.parametrize("drafted", ["chain", "tree", "draft"])
@pytest.mark.parametrize("dtype,vocab,counts", [("fp32", 1, [1, 3]), ("fp32", 7, [0, 5, 1, 64]), ("bf16", 500, [9] * 20),
                                                ("fp16", 4096, [3, 17, 2]), ("fp32", 4097, [12] * 6), ("bf16", 100003, [4, 6]),
                                                ("fp32", 40000, [33] * 3), ("bf16", 9001, [1, 3] * 200)])
def test_verification_matches(torch_gpu, drafted, dtype, vocab, counts):
    torch = torch_gpu
    say(f"case verify {drafted} {dtype} vocab={vocab} counts={counts[:5]}")
    rng = np.random.default_rng(vocab + len(counts))
    nodes = max(counts)
    total = 0
    for _ in range(3):
        case = verify_case(torch, rng, counts, vocab, drafted, dtype, width=5 if vocab < 5000 else 0)
        op = run_verify(torch, case, nodes=nodes, vocab=vocab)
        total += int(check_verify(case, op, nodes=nodes).sum())
        check_verify(case, op, nodes=nodes)  # again on the same workspace
        assert int(op.status.item()) == 0
    say(f"  kept {total} of {3 * sum(counts)}")


def test_verification_edges(torch_gpu):
    """Tokens named twice, outside the vocabulary, parents that do not come first, uniforms of 0 and just
    below 1, one-hot targets, rows without weights, NaN and negative weights, more rows than max_nodes."""
    torch = torch_gpu
    rng = np.random.default_rng(4)
    say("case verify edges")
    case = verify_case(torch, rng, [6, 6, 6, 6], 50, "tree", "fp32")
    case["parents"][:24] = [-1, 0, 0, 0, 1, 1] * 4
    case["tokens"][1:4] = 7
    case["uniforms"][:24:6], case["uniforms"][1] = [0.0, 1 - 2.0 ** -24, 0.4, 0.6], 0.0
    case["final"][:] = [0.0, 1 - 2.0 ** -24, 0.0, 1 - 2.0 ** -24]
    hot = torch.zeros((6, 50), device="cuda")
    hot[torch.arange(6), torch.from_numpy(case["tokens"][[13, 16, 14, 15, 16, 17]]).cuda()] = 1.0
    case["probs"][12:18] = hot
    check_verify(case, run_verify(torch, case, nodes=6, vocab=50), nodes=6)
    case["tokens"][[2, 9]], case["tokens"][[0, 6]] = [-1, 50], [-5, 1 << 40]
    op = run_verify(torch, case, nodes=6, vocab=50)
    check_verify(case, op, nodes=6)
    assert int(op.status.item()) == abi.STATUS_BAD_TOKEN
    case["tokens"][[2, 9]] = 3
    case["parents"][[3, 14]] = [4, -9]
    op = run_verify(torch, case, nodes=6, vocab=50)
    check_verify(case, op, nodes=6)
    assert int(op.status.item()) == abi.STATUS_BAD_TREE
    case["parents"][[3, 14]] = 0
    case["probs"][18:24] = float("nan")
    case["probs"][6:12] = 0.0
    case["probs"][0:6, ::3] = -1.0
    op = run_verify(torch, case, nodes=6, vocab=50)
    check_verify(case, op, nodes=6)
    assert int(op.status.item()) == abi.STATUS_BAD_PROBS
    case = verify_case(torch, rng, [9, 3], 50, "tree", "fp32")
    op = run_verify(torch, case, nodes=4, vocab=50)
    check_verify(case, op, nodes=4, limit=4)
    assert int(op.status.item()) == abi.STATUS_BAD_LENGTH


def test_verification_refuses(torch_gpu):
    torch = torch_gpu
    op = kvip_amd.DraftVerifier(torch, batch=2, max_nodes=3, vocab=10, device="cuda")
    probs = torch.zeros((6, 10), device="cuda")
    good = dict(probs=probs, tokens=torch.zeros(6, dtype=torch.int64, device="cuda"),
                cu_seqlens=torch.zeros(3, dtype=torch.int32, device="cuda"), uniforms=torch.zeros(6, device="cuda"),
                final_uniforms=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        op()
    parents = torch.zeros(6, dtype=torch.int32, device="cuda")
    bad = dict(probs=[probs.double(), probs[:, :9], probs.t(), probs.cpu(), probs[:0]], tokens=[good["tokens"].int(), good["tokens"][:5]],
               cu_seqlens=[good["cu_seqlens"].long(), good["cu_seqlens"][:2]], uniforms=[good["uniforms"].double(), probs[:, 0]],
               final_uniforms=[good["uniforms"]], parents=[parents.long(), parents[:5]], draft_probs=[probs.half(), probs[:5]])
    for name, values in bad.items():
        for value in values:
            with pytest.raises(ValueError):
                op.bind(**{**good, name: value})
    with pytest.raises(ValueError):
        op.bind(**good, parents=parents, draft_probs=probs)
    tokens, kept, path = op.bind(**good)()
    assert not kept.any() and bool((tokens == -1).all()) and bool((path == -1).all())


# --- a round ---------------------------------------------------------------------------------


class Round:
    """A drafted round as a serving loop runs it: tables, turned queries, stored rows, attention, verification,
    kept rows moved together. The model around it is one matrix from outputs to probabilities."""

    def __init__(self, torch, seed, batch=3, nodes=7, heads=16, vocab=300):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.torch, self.batch, self.rows, self.vocab = torch, batch, batch * nodes + 4, vocab
        self.kv = torch.zeros((40, 128, ROW), dtype=torch.uint8, device="cuda")
        self.index = torch.randn((40, 128, 128), generator=gen, device="cuda").to(torch.float8_e4m3fn)
        self.tables = kvip_amd.PageTables(torch, batch=batch, max_context=1024, num_blocks=40, max_tokens=self.rows,
                                          device="cuda", caches=[self.kv, self.index.view(torch.uint8)])
        self.rotary = kvip_amd.Rotary(torch, rotary_dim=64, device="cuda")
        self.store = kvip_amd.KvRowStore(torch, kv_cache=self.kv, rotary=self.rotary)
        self.attention = kvip_amd.TreeAttention(torch, batch=batch, heads=heads, max_nodes=nodes, max_tokens=self.rows,
                                                max_context=1024, device="cuda")
        self.verifier = kvip_amd.DraftVerifier(torch, batch=batch, max_nodes=nodes, vocab=vocab, device="cuda")
        self.counts = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.parents = torch.full((self.rows,), -1, dtype=torch.int32, device="cuda")
        self.projected = torch.zeros((self.rows, heads, 192), dtype=torch.bfloat16, device="cuda")
        self.query = torch.zeros((self.rows, heads, 576), dtype=torch.bfloat16, device="cuda")
        self.latent = torch.zeros((self.rows, 576), dtype=torch.bfloat16, device="cuda")
        self.tokens = torch.zeros(self.rows, dtype=torch.int64, device="cuda")
        self.uniforms, self.final = torch.zeros(self.rows, device="cuda"), torch.zeros(batch, device="cuda")
        self.head = torch.randn((512, vocab), generator=gen, device="cuda") * 0.5
        self.probs = torch.zeros((self.rows, vocab), device="cuda")
        t = self.tables
        self.rotary.bind(t.positions, self.projected[..., 128:], query_out=self.query[..., 512:])
        self.store.bind(self.latent[:, :512], self.latent[:, 512:], t.slots, t.positions)
        self.attention.bind(self.query, self.kv, t.block_table, t.lengths, t.cu_seqlens, t.visible)
        self.verifier.bind(self.probs, self.tokens, t.cu_seqlens, self.uniforms, self.final, parents=self.parents)

    def inputs(self, seed, counts):
        rng = np.random.default_rng(seed)
        torch = self.torch
        self.counts.copy_(torch.tensor(counts, dtype=torch.int32))
        self.parents.copy_(torch.from_numpy(random_parents(rng, counts, self.rows)))
        for x in (self.projected, self.query, self.latent):
            x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32)))
        self.tokens.copy_(torch.from_numpy(rng.integers(0, 12, self.rows)))
        self.uniforms.copy_(torch.from_numpy(rng.random(self.rows).astype(np.float32)))
        self.final.copy_(torch.from_numpy(rng.random(self.batch).astype(np.float32)))

    def step(self):
        torch = self.torch
        self.tables.extend(self.counts, self.parents)
        self.rotary()
        self.store()
        out = self.attention()
        logits = out[:, 0].float() @ self.head
        logits[:, :12] += 3.0
        self.probs.copy_(torch.softmax(logits, 1))
        tokens, kept, path = self.verifier()
        self.tables.commit(kept, path)

    def state(self):
        t, v = self.tables, self.verifier
        return [x.clone() for x in (self.kv, self.index.view(self.torch.uint8), t.block_table, t.lengths, t.free_count, t.slots,
                                    t.positions, self.attention.output[:int(t.cu_seqlens[-1])], v.out_tokens, v.kept, v.path)]


def test_a_round_matches(torch_gpu):
    """Three rounds on growing requests, every stage against the restatement fed with the stage before."""
    torch = torch_gpu
    say("case round")
    r = Round(torch, 1)
    model = draft.Tables(3, 8, 40, r.rows)
    for seed, counts in ((1, [7, 5, 6]), (2, [4, 0, 7]), (3, [7, 7, 1])):
        r.inputs(seed, counts)
        bases = list(model.lengths)
        _, slots, positions, visible, status = model.extend(counts, r.parents.tolist())
        r.step()
        torch.cuda.synchronize()
        assert status == 0
        assert r.tables.slots.tolist() == slots and r.tables.positions.tolist() == positions
        assert r.tables.visible.tolist() == visible
        f = r.rotary.frequencies.cpu().numpy()
        rope = host(r.projected[..., 128:])
        want = draft.turned(rope, positions, f, False)
        assert np.all(np.abs(host(r.query[..., 512:]) - want) <= turn_bound(rope, f, False, 1.0, want, 2.0 ** -8))
        probs, at = host(r.probs), 0
        kept, path = r.verifier.kept.tolist(), r.verifier.path.tolist()
        codes, scales = draft.stored_rows(host(r.latent)[:, :512])
        for b, n in enumerate(counts):
            if n:
                s = slice(at, at + n)
                walk, out = draft.verify(probs[s], r.tokens[s].tolist(), r.parents[s].tolist(), None, r.uniforms[s].tolist(),
                                         float(r.final[b]))
                assert path[b][:kept[b]] == walk and r.verifier.out_tokens[b].tolist()[:kept[b]] == out
                for i, node in enumerate(walk):  # the kept tokens' rows stand together
                    p = bases[b] + i
                    row = r.kv[model.pages[b][p // 128], p % 128].cpu().numpy()
                    assert np.array_equal(row[:512], codes[at + node]) and np.array_equal(row[640:].view("<f4"), scales[at + node])
            else:
                assert kept[b] == 0
            at += n
        model.commit(kept)
        same_tables(r.tables, model)
        for op in (r.tables, r.store, r.attention, r.verifier):
            assert int(op.status.item()) == 0


def test_a_captured_round_replays(torch_gpu):
    """The round captured into a graph, replayed on new inputs with eager work and synchronisations in
    between, against a second engine that runs every round eagerly, on a stream of its own."""
    torch = torch_gpu
    say("case captured round")
    eager, graphed = Round(torch, 5), Round(torch, 5)
    plan = [(s, [int(x) for x in np.random.default_rng(s).integers(0, 8, 3)]) for s in range(7)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for r in (eager, graphed):
            r.inputs(*plan[0])
            r.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        graphed.step()
    for seed, counts in plan[1:]:
        for r in (eager, graphed):
            r.inputs(seed, counts)
        eager.step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.state(), graphed.state()):
            assert torch.equal(a, b), seed


def test_calls_take_the_current_stream(torch_gpu):
    torch = torch_gpu
    device, side = torch.device("cuda", torch.cuda.current_device()), torch.cuda.Stream()
    assert abi.raw_stream(torch, device) == abi.stream_handle(torch, device)
    with torch.cuda.stream(side):
        assert abi.raw_stream(torch, device) == abi.stream_handle(torch, device) == side.cuda_stream


def test_objects_run_side_by_side(torch_gpu):
    """Two engines on two streams at once do not touch one another's workspaces."""
    torch = torch_gpu
    say("case two streams")
    alone, a, b = Round(torch, 7), Round(torch, 7), Round(torch, 7)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in range(4):
        for r in (alone, a, b):
            r.inputs(seed, [7, 6, 5])
        alone.step()
        torch.cuda.synchronize()
        for r, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                r.step()
        torch.cuda.synchronize()
        for x, y, z in zip(alone.state(), a.state(), b.state()):
            assert torch.equal(x, y) and torch.equal(x, z)
