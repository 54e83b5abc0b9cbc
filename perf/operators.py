"""Performance cases of the operators of a round of drafted tokens over the paged KV rows: the
calls a serving engine makes when every request brings a few drafted tokens (a chain or a tree).

Kinds of case:
  tables   kvip_amd.PageTables: pages, slots, positions and visibility of a step's tokens from the
           request lengths, and the same pages given back when no token is kept (so that a pass
           ends where it began).
  rotary   kvip_amd.Rotary: the rotary part of queries and keys turned by their positions.
  store    kvip_amd.KvRowStore: latents quantised to 656-byte rows, their rotary features turned,
           written to the tokens' slots.
  tree     kvip_amd.TreeAttention: every step token of every request attends its whole context
           and those step tokens that its visibility names.
  verify   kvip_amd.DraftVerifier: drafted tokens accepted or refused against the target's
           probabilities by given random numbers, and the token that follows the last accepted one.

Request lengths follow from the case alone, so that every seed gives the same shapes; values,
tables, trees and random numbers follow from the seed.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
BLOCK = 128
KEY_DIM, VALUE_DIM, ROPE_DIM, ROW_BYTES = 576, 512, 64, 656
_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One interactive request, 16 of 128 heads (8-way tensor parallel): latency counts.
        _tree("tree_single", batch=1, heads=16, nodes=6, ctx_low=900, ctx_high=900),
        # The benchmark's decode batch with one token and its three drafted ones per request.
        _tree("tree_b64_h16", batch=64, heads=16, nodes=4, ctx_low=1000, ctx_high=16384),
        # All 128 heads and wider trees on fewer requests: the matrix products count.
        _tree("tree_b8_h128", batch=8, heads=128, nodes=12, ctx_low=2000, ctx_high=8192),
        # Two very long contexts (history of the repository's long-context configuration).
        _tree("tree_128k", batch=2, heads=32, nodes=9, ctx_low=100000, ctx_high=131000),
        # The same step's query and key heads before they meet the cache, interleaved pairs.
        _rotary("rotary_step", tokens=256, heads=16, dim=64, rotary=64, layout="interleaved", scaling="none", dtype="bf16",
                top=32768),
        # The index queries of a long prompt: half of each head turned, halves layout, stretched context.
        _rotary("rotary_prompt", tokens=8192, heads=64, dim=128, rotary=64, layout="half", scaling="yarn", dtype="bf16",
                top=131072),
        # The rows of one step of 64 requests of four tokens.
        _store("store_step", tokens=256, layout="interleaved", scaling="none", top=32768),
        # The rows of prompts.
        _store("store_prompt", tokens=20000, layout="half", scaling="yarn", top=131072),
        # A step of 64 requests with small trees.
        _tables("tables_step", batch=64, count_low=1, count_high=9, ctx_low=100, ctx_high=32768, trees=True),
        # The largest step: prompt chunks of many requests.
        _tables("tables_prompt", batch=300, count_low=1, count_high=700, ctx_low=0, ctx_high=65536, trees=False),
        # Trees of chosen tokens on a few requests.
        _verify("verify_tree", batch=16, count_low=5, count_high=17, vocab=32000, drafted="tree", dtype="fp32"),
        # Chains drawn from a draft distribution, a large vocabulary.
        _verify("verify_chain", batch=64, count_low=5, count_high=5, vocab=131072, drafted="chain", dtype="fp32"),
    ]


def _tree(name, *, batch, heads, nodes, ctx_low, ctx_high):
    return _named(name, kind="tree", batch=batch, heads=heads, nodes=nodes, ctx_low=ctx_low, ctx_high=ctx_high)


def _rotary(name, *, tokens, heads, dim, rotary, layout, scaling, dtype, top):
    return _named(name, kind="rotary", tokens=tokens, heads=heads, dim=dim, rotary=rotary, layout=layout, scaling=scaling,
                  dtype=dtype, top=top)


def _store(name, *, tokens, layout, scaling, top):
    return _named(name, kind="store", tokens=tokens, layout=layout, scaling=scaling, top=top)


def _tables(name, *, batch, count_low, count_high, ctx_low, ctx_high, trees):
    return _named(name, kind="tables", batch=batch, count_low=count_low, count_high=count_high, ctx_low=ctx_low,
                  ctx_high=ctx_high, trees=trees)


def _verify(name, *, batch, count_low, count_high, vocab, drafted, dtype):
    return _named(name, kind="verify", batch=batch, count_low=count_low, count_high=count_high, vocab=vocab,
                  drafted=drafted, dtype=dtype)


def _named(name, **case):
    return case if name is None else {"name": name, **case}


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "rotary", "rotary", "store", "tables", "verify", "verify"])
    if kind == "tree":
        heads = rng.choice([8, 16, 20, 32, 64, 128])
        nodes = _log(rng, 1, 33)
        batch = _log(rng, 1, 96)
        # At most the work of the largest listed cases: products and bytes.
        top = min(131000, 50_000_000 // (batch * nodes * heads) + 64, 560_000 // batch)
        high = _log(rng, 64, max(64, top))
        return _tree(None, batch=batch, heads=heads, nodes=nodes, ctx_low=_log(rng, 1, high), ctx_high=high)
    if kind == "rotary":
        rotary = rng.choice([32, 64, 64, 128])
        heads = rng.choice([1, 8, 16, 20, 64, 128])
        dim = rng.choice([rotary, 128 if rotary < 128 else 192])
        return _rotary(None, tokens=_log(rng, 1, 8192 * 64 * 128 // (2 * heads * dim)), heads=heads, dim=dim, rotary=rotary,
                       layout=rng.choice(["interleaved", "half"]), scaling=rng.choice(["none", "linear", "yarn"]),
                       dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), top=_log(rng, 100, 1 << 20))
    if kind == "store":
        return _store(None, tokens=_log(rng, 1, 20000), layout=rng.choice(["interleaved", "half"]),
                      scaling=rng.choice(["none", "yarn"]), top=_log(rng, 100, 1 << 20))
    if kind == "tables":
        batch, trees = _log(rng, 1, 300), rng.random() < 0.6
        high = _log(rng, 1, 64) if trees else _log(rng, 1, 700)
        ctx = _log(rng, 1, 65536)
        return _tables(None, batch=batch, count_low=rng.randint(0, high), count_high=high, ctx_low=rng.randint(0, ctx),
                       ctx_high=ctx, trees=trees)
    drafted = rng.choice(["tree", "chain"])
    vocab = _log(rng, 500, 131072)
    high = _log(rng, 1, 33 if drafted == "tree" else 9)
    batch = _log(rng, 1, max(1, min(128, 40_000_000 // (vocab * high))))
    return _verify(None, batch=batch, count_low=rng.randint(1, high), count_high=high, vocab=vocab, drafted=drafted,
                   dtype=rng.choice(["fp32", "fp32", "bf16"]))


# --- inputs -------------------------------------------------------------------------------


def prepare(case, seed):
    return {"tree": _prepare_tree, "rotary": _prepare_rotary, "store": _prepare_store, "tables": _prepare_tables,
            "verify": _prepare_verify}[case["kind"]](case, seed)


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE)


def _device(values, dtype):
    return torch.from_numpy(np.ascontiguousarray(values)).to(dtype).to(DEVICE)


def _spread(low, high, count):
    """Whole numbers between low and high, the first of them high, spread evenly in no order."""
    return np.asarray([high - int((i * 0.6180339887498949 % 1.0) * (high - low + 1)) for i in range(count)], np.int64)


def _kv_rows(gen, count):
    """uint8 [count, 656]: 512 fp8 features of N(0, 1) values with one scale per 128, 64 bf16
    rope features, the four scales."""
    rows = torch.empty((count, ROW_BYTES), dtype=torch.uint8, device=DEVICE)
    for at in range(0, count, 1 << 17):
        part = rows[at:at + (1 << 17)]
        values = _normal(gen, len(part), 4, 128)
        scales = values.abs().amax(2) / 448
        part[:, :512] = (values / scales[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).view(-1, 512)
        part[:, 512:640] = _normal(gen, len(part), 64).to(torch.bfloat16).view(torch.uint8)
        part[:, 640:] = scales.view(torch.uint8)
    return rows


def _trees(rng, counts):
    """Parents (within the request, -1 for the root) of every step token."""
    parents = []
    for n in counts:
        parents += [-1 if i == 0 else int(rng.integers(max(0, i - 4), i)) for i in range(n)]
    return np.asarray(parents, np.int32)


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)])


def _seen(parents, counts):
    """Visibility bits of every step token: itself and its ancestors, as its request's tokens."""
    bits, at = np.zeros(len(parents), np.uint64), 0
    for n in counts:
        for i in range(n):
            own_bit, up = np.uint64(1) << np.uint64(i), parents[at + i]
            bits[at + i] = own_bit | (bits[at + up] if up >= 0 else np.uint64(0))
        at += n
    return bits.view(np.int64)


def _prepare_tree(case, seed):
    gen, rng = _generator(seed), np.random.default_rng(seed)
    batch, heads, nodes = case["batch"], case["heads"], case["nodes"]
    counts = np.full(batch, nodes, np.int64)
    lens = _spread(case["ctx_low"], case["ctx_high"], batch) + counts
    blocks = -(-lens // BLOCK)
    pages = int(blocks.sum())
    kv = _kv_rows(gen, pages * BLOCK).view(pages, BLOCK, ROW_BYTES)
    table, at, order = np.full((batch, int(blocks.max())), -1, np.int32), 0, rng.permutation(pages)
    for b, n in enumerate(blocks):
        table[b, :n] = order[at:at + n]
        at += n
    state = {"kind": "tree", "kv": kv, "table": _device(table, torch.int32), "lens": _device(lens, torch.int32),
             "starts": _device(_starts(counts), torch.int32),
             "seen": _device(_seen(_trees(rng, counts), counts), torch.int64),
             "query": _normal(gen, batch * nodes, heads, KEY_DIM).to(torch.bfloat16), "nodes": nodes, "top": int(lens.max())}
    if own:
        import kvip_amd

        op = kvip_amd.TreeAttention(torch, batch=batch, heads=heads, max_nodes=nodes, max_tokens=batch * nodes,
                                    max_context=int(lens.max()), device=DEVICE)
        state["op"] = op.bind(state["query"], kv, state["table"], state["lens"], state["starts"], state["seen"])
    return state


def _frequencies(rotary, scaling):
    """Angle per position of each of the rotary / 2 pairs, and what the result is multiplied by."""
    plain = [10000.0 ** (-2.0 * i / rotary) for i in range(rotary // 2)]
    if scaling["kind"] == "linear":
        return [f / scaling["factor"] for f in plain], 1.0
    if scaling["kind"] == "yarn":
        def turns_at(turns):  # the pair that turns so often over the original context
            return rotary * math.log(scaling["original"] / (turns * 2 * math.pi)) / (2 * math.log(10000.0))

        low = max(math.floor(turns_at(scaling["beta_fast"])), 0)
        high = min(math.ceil(turns_at(scaling["beta_slow"])), rotary - 1)
        keep = [1.0 - min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(rotary // 2)]
        return ([f * k + f / scaling["factor"] * (1.0 - k) for f, k in zip(plain, keep)],
                0.1 * math.log(scaling["factor"]) + 1.0)
    return plain, 1.0


_SCALINGS = {"none": {"kind": "none"}, "linear": {"kind": "linear", "factor": 4.0},
             "yarn": {"kind": "yarn", "factor": 40.0, "original": 4096, "beta_fast": 32.0, "beta_slow": 1.0}}


def _angles(state, case, rotary):
    frequencies, factor = _frequencies(rotary, _SCALINGS[case["scaling"]])
    state.update(frequencies=torch.tensor(frequencies, dtype=torch.float64, device=DEVICE), factor=factor,
                 half=case["layout"] == "half", rotary=rotary)


def _positions(gen, count, top):
    return torch.randint(0, top, (count,), generator=gen, device=DEVICE)


def _rotary_op(case, rotary):
    import kvip_amd

    scaling = _SCALINGS[case["scaling"]]
    return kvip_amd.Rotary(torch, rotary_dim=rotary, layout=case["layout"],
                           scaling=None if scaling["kind"] == "none" else scaling, device=DEVICE)


def _prepare_rotary(case, seed):
    gen, dtype = _generator(seed), _DTYPES[case["dtype"]]
    tokens, heads, dim = case["tokens"], case["heads"], case["dim"]
    # The part to turn is a slice of what the projection wrote, and goes into a slice of the query.
    state = {"kind": "rotary", "positions": _positions(gen, tokens, case["top"]),
             "query": _normal(gen, tokens, heads, 64 + dim).to(dtype)[..., 64:],
             "key": _normal(gen, tokens, VALUE_DIM + dim).to(dtype)[:, VALUE_DIM:],
             "query_out": torch.zeros((tokens, heads, dim + 64), dtype=dtype, device=DEVICE)[..., 64:],
             "key_out": torch.zeros((tokens, dim), dtype=dtype, device=DEVICE)}
    _angles(state, case, case["rotary"])
    if own:
        state["op"] = _rotary_op(case, case["rotary"]).bind(state["positions"], state["query"], state["key"],
                                                            query_out=state["query_out"], key_out=state["key_out"])
    return state


def _prepare_store(case, seed):
    gen, tokens = _generator(seed), case["tokens"]
    pages = 2 * -(-tokens // BLOCK)
    # Latent and rotary features come from one projection.
    projected = _normal(gen, tokens, KEY_DIM).to(torch.bfloat16)
    state = {"kind": "store", "latent": projected[:, :VALUE_DIM], "rope": projected[:, VALUE_DIM:],
             "kv": _kv_rows(gen, pages * BLOCK).view(pages, BLOCK, ROW_BYTES),
             "slots": torch.randperm(pages * BLOCK, generator=gen, device=DEVICE)[:tokens].contiguous(),
             "positions": _positions(gen, tokens, case["top"])}
    state["slots"][tokens // 2::97] = -1  # padded tokens
    _angles(state, case, ROPE_DIM)
    if own:
        import kvip_amd

        op = kvip_amd.KvRowStore(torch, kv_cache=state["kv"], rotary=_rotary_op(case, ROPE_DIM))
        state["op"] = op.bind(state["latent"], state["rope"], state["slots"], state["positions"])
    return state


def _prepare_tables(case, seed):
    rng = np.random.default_rng(seed)
    batch = case["batch"]
    counts = _spread(case["count_low"], case["count_high"], batch)
    lens = _spread(case["ctx_low"], case["ctx_high"], batch)[::-1].copy()
    tokens = int(counts.sum()) + 5  # a few rows behind the last token, as a padded step has
    held, need = -(-lens // BLOCK), -(-(lens + counts) // BLOCK)
    pages = int(need.sum()) + 64
    width = -(-(case["ctx_high"] + case["count_high"]) // BLOCK)
    order = rng.permutation(pages).astype(np.int32)
    table, at = np.full((batch, width), -1, np.int32), 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    free = np.full(pages, -1, np.int32)
    free[:pages - at] = order[at:]
    state = {"kind": "tables", "counts": _device(counts, torch.int32), "lengths": _device(lens, torch.int32),
             "table": _device(table, torch.int32), "free": _device(free, torch.int32),
             "free_count": torch.tensor([pages - at], dtype=torch.int32, device=DEVICE), "tokens": tokens,
             "parents": None, "most": case["count_high"]}
    if case["trees"]:
        parents = np.full(tokens, -1, np.int32)
        parents[:tokens - 5] = _trees(rng, counts)
        state["parents"] = _device(parents, torch.int32)
    if own:
        import kvip_amd

        op = kvip_amd.PageTables(torch, batch=batch, max_context=width * BLOCK, num_blocks=pages, max_tokens=tokens,
                                 device=DEVICE)
        op.block_table.copy_(state["table"])
        op.lengths.copy_(state["lengths"])
        op.free.copy_(state["free"])
        op.free_count.copy_(state["free_count"])
        state["op"] = op
    return state


def _prepare_verify(case, seed):
    gen, rng = _generator(seed), np.random.default_rng(seed)
    batch, vocab, dtype = case["batch"], case["vocab"], _DTYPES[case["dtype"]]
    counts = _spread(case["count_low"], case["count_high"], batch)
    total, starts = int(counts.sum()), _starts(counts)
    logits = 5.0 * _normal(gen, total, vocab)
    state = {"kind": "verify", "starts": _device(starts, torch.int32), "nodes": int(counts.max()), "draft": None,
             "parents": None, "seen": None, "probs": torch.softmax(logits, 1).to(dtype),
             "uniforms": torch.rand(total, generator=gen, device=DEVICE),
             "final": torch.rand(batch, generator=gen, device=DEVICE)}
    if case["drafted"] == "chain":
        draft = torch.softmax(logits + 0.7 * _normal(gen, total, vocab), 1).to(dtype)
        drawn = torch.multinomial(draft.float(), 1, generator=gen)[:, 0]
        state.update(draft=draft, tokens=torch.roll(drawn, 1).contiguous())  # row i's draft is row i + 1's token
    else:
        parents = _trees(rng, counts)
        rank = np.zeros(total, np.int64)  # the how-manieth child of its parent a token is
        up = np.arange(total)
        for s, n in zip(starts[:-1], counts):
            seen = {}
            for i in range(1, n):
                p = int(parents[s + i])
                rank[s + i], up[s + i], seen[p] = seen.get(p, 0), s + p, seen.get(p, 0) + 1
        best = logits.topk(min(8, vocab), 1).indices
        state.update(parents=_device(parents, torch.int32), seen=_device(_seen(parents, counts), torch.int64),
                     tokens=best[_device(up, torch.int64), _device(rank % min(8, vocab), torch.int64)])
    del logits
    if own:
        import kvip_amd

        op = kvip_amd.DraftVerifier(torch, batch=batch, max_nodes=state["nodes"], vocab=vocab, device=DEVICE)
        state["op"] = op.bind(state["probs"], state["tokens"], state["starts"], state["uniforms"], state["final"],
                              parents=state["parents"], draft_probs=state["draft"])
    return state


# --- one pass -----------------------------------------------------------------------------


def run(state):
    if own:
        return {"tree": _own_tree, "rotary": _own_rotary, "store": _own_store, "tables": _own_tables,
                "verify": _own_verify}[state["kind"]](state)
    return {"tree": _plain_tree, "rotary": _plain_rotary, "store": _plain_store, "tables": _plain_tables,
            "verify": _plain_verify}[state["kind"]](state)


def _own_tree(state):
    return [state["op"]()]


def _own_rotary(state):
    state["op"]()
    return [state["query_out"], state["key_out"]]


def _own_store(state):
    state["op"]()
    return _parts(state["kv"])


def _own_tables(state):
    op = state["op"]
    op.extend(state["counts"], state["parents"])
    op.truncate(state["lengths"])
    outputs = [op.cu_seqlens, op.positions, op.slots, op.block_table, op.lengths, op.free, op.free_count]
    return outputs + ([op.visible] if state["parents"] is not None else [])


def _own_verify(state):
    return list(state["op"]())


# --- the plain forms ----------------------------------------------------------------------


def _padded(starts, count, nodes):
    """Row numbers [batch, nodes] of a packed step, and which of them exist."""
    at = torch.arange(nodes, device=DEVICE)
    rows = starts[:-1].long()[:, None] + at
    live = rows < starts[1:].long()[:, None]
    return rows.clamp(max=count - 1), live


def _plain_tree(s):
    """softmax(scale * q k) v in 32 bits over every cached row of the request, step tokens by their bits."""
    batch, nodes, heads, top = len(s["lens"]), s["nodes"], s["query"].shape[1], s["top"]
    at = torch.arange(top, device=DEVICE)
    pages = s["table"][:, at // BLOCK].long().clamp(min=0)
    raw = s["kv"][pages, at % BLOCK]
    nope = raw[..., :VALUE_DIM].contiguous().view(torch.float8_e4m3fn).float().view(batch, top, 4, 128)
    value = (nope * raw[..., 640:].contiguous().view(torch.float32)[..., None]).view(batch, top, VALUE_DIM)
    key = torch.cat([value, raw[..., 512:640].contiguous().view(torch.bfloat16).float()], -1)
    past = s["lens"][:, None, None].long() - nodes
    bits = s["seen"].view(batch, nodes)[:, :, None] >> (at - past).clamp(0, 63)
    sees = (at < past) | ((at < past + nodes) & ((bits & 1) == 1))
    query = s["query"].float().view(batch, nodes * heads, KEY_DIM)
    logits = torch.matmul(query, key.transpose(1, 2).contiguous()).view(batch, nodes, heads, top) * KEY_DIM ** -0.5
    logits = logits.masked_fill(~sees[:, :, None, :], float("-inf"))
    weight = torch.exp(logits - logits.amax(-1, keepdim=True))
    weight = (weight / weight.sum(-1, keepdim=True)).view(batch, nodes * heads, top)
    return [torch.matmul(weight, value).view(batch * nodes, heads, VALUE_DIM).to(torch.bfloat16)]


def _turned(x, s):
    """x [tokens, ..., dim] with its first features turned by the tokens' angles, in 32 bits."""
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = ((f(angle) * s["factor"]).float() for f in (torch.cos, torch.sin))
    shape = (len(x),) + (1,) * (x.dim() - 2) + (s["rotary"] // 2,)
    cos, sin, part = cos.view(shape), sin.view(shape), x[..., :s["rotary"]].float()
    if s["half"]:
        a, b = part.chunk(2, -1)
        part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([part, x[..., s["rotary"]:].float()], -1).to(x.dtype)


def _plain_rotary(s):
    return [_turned(s["query"], s), _turned(s["key"], s)]


def _parts(kv):
    """The features, rotary features and scales that the cache's rows hold."""
    return [kv[..., :512].view(torch.float8_e4m3fn), kv[..., 512:640].view(torch.bfloat16),
            kv[..., 640:656].view(torch.float32)]


def _plain_store(s):
    tokens = len(s["slots"])
    kept = s["slots"] >= 0
    parts = s["latent"].float().view(tokens, 4, 128)
    largest = parts.abs().amax(2)
    scales = torch.where(largest > 0, largest / 448, torch.ones_like(largest))
    nope = (parts / scales[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(tokens, 512)
    rows = torch.cat([nope.view(torch.uint8), _turned(s["rope"], s).contiguous().view(torch.uint8),
                      scales.view(torch.uint8)], 1)
    s["kv"].view(-1, ROW_BYTES)[s["slots"][kept]] = rows[kept]
    return _parts(s["kv"])


def _plain_tables(s):
    lengths, counts, table, free = s["lengths"].long(), s["counts"].long(), s["table"], s["free"]
    held, after = -(-lengths // BLOCK), -(-(lengths + counts) // BLOCK)
    need = after - held
    first = torch.cumsum(need, 0) - need
    column = torch.arange(table.shape[1], device=DEVICE)[None, :]
    fresh = (column >= held[:, None]) & (column < after[:, None])
    taken = (s["free_count"].long() - 1 - (first[:, None] + column - held[:, None])).clamp(0, len(free) - 1)
    table = torch.where(fresh, free[taken], table)
    ends = torch.cumsum(counts, 0)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends])
    token = torch.arange(s["tokens"], device=DEVICE)
    request = torch.searchsorted(ends, token, right=True).clamp(max=len(counts) - 1)
    live, within = token < ends[-1], token - cu[request]
    at = lengths[request] + within
    slots = torch.where(live, table[request, (at // BLOCK).clamp(max=table.shape[1] - 1)].long() * BLOCK + at % BLOCK, -1)
    outputs, depth = [], within
    if s["parents"] is not None:
        n = s["most"]
        rows, there = _padded(cu, s["tokens"], n)
        up = torch.where(there, s["parents"][rows].long(), -1)
        node = torch.arange(n, device=DEVICE)
        closed = (up[:, :, None] == node).float() + torch.eye(n, device=DEVICE)
        closed = (torch.matrix_power(closed, 64) > 0) & there[:, :, None]  # a tree of 64 tokens is at most 64 deep
        bits = (closed.long() << node).sum(-1)
        seen, deep = torch.zeros(s["tokens"], dtype=torch.int64, device=DEVICE), torch.zeros_like(token)
        seen[rows[there]], deep[rows[there]] = bits[there], closed.sum(-1)[there] - 1
        outputs, depth = [seen], deep
    positions = torch.where(live, lengths[request] + depth, 0)
    # Nothing is kept: the pages go back in the order that undoes their taking.
    back = torch.where(fresh, s["free_count"].long() - 1 - (first[:, None] + column - held[:, None]), len(free))
    stack = torch.cat([free, free[:1]]).scatter(0, back.clamp(max=len(free)).view(-1), table.view(-1))[:-1]
    table = torch.where(column < held[:, None], table, torch.full_like(table, -1))
    return [cu.int(), positions, slots, table, lengths.int(), stack, s["free_count"].clone()] + outputs


def _drawn(weights, uniforms):
    """The first place of each row at which its running sum passes the uniform's share of the whole."""
    run = torch.cumsum(weights, 1)
    return torch.searchsorted(run, (uniforms.double() * run[:, -1])[:, None], right=True)[:, 0].clamp(max=weights.shape[1] - 1)


def _plain_verify(s):
    probs, tokens, nodes = s["probs"], s["tokens"].long(), s["nodes"]
    rows, live = _padded(s["starts"], len(tokens), nodes)
    batch, node = len(rows), torch.arange(nodes, device=DEVICE)
    names = tokens[rows]
    if s["draft"] is not None:
        after = rows[:, 1:]  # the token that each row but the last drafted
        taken = s["uniforms"][rows[:, :-1]].double() * s["draft"][rows[:, :-1], tokens[after]].double() < \
            probs[rows[:, :-1], tokens[after]].double()
        path = torch.cat([torch.ones_like(live[:, :1]), torch.cumprod((taken & live[:, 1:]).long(), 1).bool()], 1)
    else:
        up = s["parents"][rows].long()
        child = (up >= 0) & live
        value = torch.where(child, probs[rows.gather(1, up.clamp(min=0)), names].double(), 0.0)
        before = (up[:, :, None] == up[:, None, :]) & child[:, :, None] & child[:, None, :] & (node[None, :] < node[:, None])
        again = (before & (names[:, :, None] == names[:, None, :])).any(2)
        value = value.masked_fill(again, 0.0)  # a token named before has nothing left
        low = (before * value[:, None, :]).sum(2)
        u = s["uniforms"][rows.gather(1, up.clamp(min=0))].double()
        chosen = (child & (low <= u) & (u < low + value)) | (node == 0)
        above = (s["seen"][rows][:, :, None] >> node) & 1
        path = live & ((above == 0) | chosen[:, None, :]).all(2)
    kept = path.sum(1)
    order = torch.where(path, node, nodes).sort(1).values
    last = order.gather(1, (kept - 1)[:, None])
    here = rows.gather(1, last)[:, 0]
    rest = probs[here].double()
    if s["draft"] is not None:
        refused = here + 1 < s["starts"][1:].long()
        rest = torch.where(refused[:, None], (rest - s["draft"][here].double()).clamp(min=0), rest)
    else:
        tried = child & (up == last)
        gone = torch.zeros((batch, rest.shape[1] + 1), dtype=torch.bool, device=DEVICE)
        gone.scatter_(1, torch.where(tried, names, rest.shape[1]), True)
        rest = rest.masked_fill(gone[:, :-1], 0.0)
    final = _drawn(rest, s["final"])
    path = torch.where(node < kept[:, None], order, -1)
    following = torch.where(node + 1 < kept[:, None], names.gather(1, torch.roll(path, -1, 1).clamp(min=0)), -1)
    following = torch.where(node + 1 == kept[:, None], final[:, None], following)
    return [following, kept.int(), path.int()]


# --- the operators in 64 bits -------------------------------------------------------------


def exact(case, seed):
    if case["kind"] in ("tables", "verify"):
        return None  # whole numbers
    state = prepare(case, seed)
    return {"tree": _exact_tree, "rotary": _exact_rotary, "store": _exact_store}[case["kind"]](state)


def _exact_tree(s):
    out, nodes = [], s["nodes"]
    for b, length in enumerate(s["lens"].tolist()):
        rows = s["kv"][s["table"][b, :-(-length // BLOCK)].long()].reshape(-1, ROW_BYTES)[:length].contiguous()
        scale = rows[:, 640:656].contiguous().view(torch.float32).double().repeat_interleave(128, 1)
        value = rows[:, :512].contiguous().view(torch.float8_e4m3fn).double() * scale
        key = torch.cat([value, rows[:, 512:640].contiguous().view(torch.bfloat16).double()], 1).t().contiguous()
        for i in range(nodes):
            bits = int(s["seen"][b * nodes + i])
            hidden = [length - nodes + j for j in range(nodes) if not bits >> j & 1]
            logits = s["query"][b * nodes + i].double() @ key / math.sqrt(KEY_DIM)
            logits[:, hidden] = -math.inf
            out.append(torch.softmax(logits, 1) @ value)
    return [torch.stack(out)]


def _exact_turn(x, s):
    """Each pair as a complex number times e^(i angle)."""
    r = s["rotary"]
    angle = torch.outer(s["positions"].double(), s["frequencies"])
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)
    turn = turn.reshape((len(x),) + (1,) * (x.dim() - 2) + (r // 2,))
    y = x.double()
    pairs = torch.complex(y[..., :r // 2], y[..., r // 2:r]) if s["half"] else \
        torch.complex(y[..., 0:r:2].contiguous(), y[..., 1:r:2].contiguous())
    pairs = pairs * turn
    y = y.clone()
    if s["half"]:
        y[..., :r // 2], y[..., r // 2:r] = pairs.real, pairs.imag
    else:
        y[..., 0:r:2], y[..., 1:r:2] = pairs.real, pairs.imag
    return y


def _exact_rotary(s):
    return [_exact_turn(s["query"], s), _exact_turn(s["key"], s)]


def _exact_store(s):
    nope, rope, scales = (p.double() for p in _parts(s["kv"]))
    nope, rope, scales = nope.view(-1, 512), rope.view(-1, 64), scales.view(-1, 4)
    at = s["slots"][s["slots"] >= 0]
    latent = s["latent"][s["slots"] >= 0].double().view(-1, 4, 128)
    scale = latent.abs().amax(2) / 448
    scale[scale == 0] = 1.0
    y = latent / scale[:, :, None]
    # e4m3: steps of 2^(exponent - 3), the exponent at least -6; halves to the even step.
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
    nope[at], scales[at] = (torch.round(y / step) * step).view(-1, 512), scale
    rope[at] = _exact_turn(s["rope"], s)[s["slots"] >= 0]
    shape = s["kv"].shape[:2]
    return [nope.view(*shape, 512), rope.view(*shape, 64), scales.view(*shape, 4)]


# --- what a pass cannot do without --------------------------------------------------------


def work(case):
    """Bytes of every input read once and every output written once, and the operations."""
    kind = case["kind"]
    if kind == "tree":
        batch, heads, nodes = case["batch"], case["heads"], case["nodes"]
        tokens = int(_spread(case["ctx_low"], case["ctx_high"], batch).sum()) + batch * nodes
        rows = batch * nodes * heads
        return {"bytes": tokens * (ROW_BYTES + 4 / BLOCK) + rows * (KEY_DIM + VALUE_DIM) * 2 + batch * (8 + 8 * nodes),
                "flops": 2.0 * (KEY_DIM + VALUE_DIM) * nodes * heads * tokens}
    if kind == "rotary":
        values = case["tokens"] * (case["heads"] + 1) * case["dim"]
        width = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2.0 * values * width + 8 * case["tokens"],
                "flops": 3.0 * case["tokens"] * (case["heads"] + 1) * case["rotary"]}
    if kind == "store":
        return {"bytes": case["tokens"] * (KEY_DIM * 2 + ROW_BYTES + 16.0), "flops": 3.0 * case["tokens"] * KEY_DIM}
    if kind == "tables":
        counts = _spread(case["count_low"], case["count_high"], case["batch"])
        lens = _spread(case["ctx_low"], case["ctx_high"], case["batch"])[::-1]
        fresh, tokens = int((-(-(lens + counts) // BLOCK) + -lens // BLOCK).sum()), int(counts.sum()) + 5
        # Taken: a page read and its entry written; given back: the entry read and cleared, the page written.
        return {"bytes": 20.0 * fresh + tokens * (28 if case["trees"] else 16) + 24 * case["batch"] + 20,
                "flops": 8.0 * tokens}
    counts = _spread(case["count_low"], case["count_high"], case["batch"])
    width = 4 if case["dtype"] == "fp32" else 2
    rows = case["vocab"] * width * (2 if case["drafted"] == "chain" else 1)  # the row that the last token is drawn from
    return {"bytes": case["batch"] * (rows + 12.0 + 12 * int(counts.max())) + int(counts.sum()) * 24.0,
            "flops": 3.0 * case["batch"] * case["vocab"]}
