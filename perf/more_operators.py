"""Performance cases of the operators on either side of a prompt chunk's layers: what a serving engine
calls when it takes a chunk of a prompt through the paged cache, and when it turns logits into the
probabilities that a token is drawn from or drafted tokens are verified against.

Kinds of case:
  chunk    kvip_amd.ChunkAttention: every token of a chunk (any number of them per request, from one up)
           attends its request's cached rows up to its own, read through the block table.
  norm     kvip_amd.NormRotary: queries and keys normed per head and turned by their positions in one
           pass; the indexer's as fp8 with one scale per head, its keys into their paged cache.
  logits   kvip_amd.LogitProcessor: penalties for repeated tokens, biases and grammar masks on logits,
           temperature, probabilities.
  history  kvip_amd.TokenHistory: which tokens admitted requests hold already, and how often.

Request lengths follow from the case alone, so that every seed gives the same shapes; values, tables, tokens,
trees and masks follow from the seed.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
BLOCK = 128
KEY_DIM, VALUE_DIM, ROW_BYTES, INDEX_DIM = 576, 512, 656, 128
EPSILON = 1e-6
_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One interactive request, 16 of 128 heads (8-way tensor parallel), the end of its prompt: latency counts.
        _chunk("chunk_single", batch=1, heads=16, count_low=130, count_high=130, ctx_low=900, ctx_high=900),
        # Ragged prompt chunks and decoding requests (one token) of one batch.
        _chunk("chunk_mixed", batch=12, heads=16, count_low=1, count_high=700, ctx_low=0, ctx_high=16000),
        # All 128 heads on a chunk of 2048 tokens.
        _chunk("chunk_h128", batch=1, heads=128, count_low=2048, count_high=2048, ctx_low=6144, ctx_high=6144),
        # The last chunk of a long prompt: 4096 tokens against 65536 rows (the repository's long-prompt configuration).
        _chunk("chunk_64k", batch=1, heads=16, count_low=4096, count_high=4096, ctx_low=61440, ctx_high=61440),
        # The indexer's inputs in a decode step of 64 requests with four tokens: queries turned, keys normed.
        _norm("norm_index_step", tokens=256, heads=64, keys=1, dim=128, rotary=64, layout="half", scaling="yarn",
              query_norm=None, key_norm="layer", index=True, dtype="bf16", top=32768),
        # The same for a prompt chunk of 8192 tokens.
        _norm("norm_index_prompt", tokens=8192, heads=64, keys=1, dim=128, rotary=64, layout="half", scaling="yarn",
              query_norm=None, key_norm="layer", index=True, dtype="bf16", top=131072),
        # Queries and keys of grouped heads, both normed, whole heads turned, in the type they came in.
        _norm("norm_heads", tokens=4001, heads=32, keys=8, dim=128, rotary=128, layout="half", scaling="none",
              query_norm="rms", key_norm="rms", index=False, dtype="bf16", top=32768),
        # One request's next token over a large vocabulary: latency counts.
        _logits("logits_single", batch=1, rows_low=1, rows_high=1, vocab=131072, past_low=1500, past_high=1500, biases=20,
                masked=False, dtype="fp32"),
        # A verified step of 64 requests with four drafted tokens each.
        _logits("logits_chain", batch=64, rows_low=5, rows_high=5, vocab=131072, past_low=200, past_high=16384, biases=0,
                masked=False, dtype="bf16"),
        # Trees of constrained requests: a grammar mask per row, biases per request.
        _logits("logits_grammar", batch=16, rows_low=5, rows_high=17, vocab=32000, past_low=100, past_high=4000, biases=64,
                masked=True, dtype="fp32"),
        # Two requests come in.
        _history("history_two", batch=2, past_low=300, past_high=900, vocab=32000),
        # A batch is filled with requests of long prompts.
        _history("history_batch", batch=32, past_low=1000, past_high=30000, vocab=131072),
    ]


def _chunk(name, *, batch, heads, count_low, count_high, ctx_low, ctx_high):
    return _named(name, kind="chunk", batch=batch, heads=heads, count_low=count_low, count_high=count_high, ctx_low=ctx_low,
                  ctx_high=ctx_high)


def _norm(name, *, tokens, heads, keys, dim, rotary, layout, scaling, query_norm, key_norm, index, dtype, top):
    return _named(name, kind="norm", tokens=tokens, heads=heads, keys=keys, dim=dim, rotary=rotary, layout=layout,
                  scaling=scaling, query_norm=query_norm or "none", key_norm=key_norm or "none", index=index, dtype=dtype, top=top)


def _logits(name, *, batch, rows_low, rows_high, vocab, past_low, past_high, biases, masked, dtype):
    return _named(name, kind="logits", batch=batch, rows_low=rows_low, rows_high=rows_high, vocab=vocab, past_low=past_low,
                  past_high=past_high, biases=biases, masked=masked, dtype=dtype)


def _history(name, *, batch, past_low, past_high, vocab):
    return _named(name, kind="history", batch=batch, past_low=past_low, past_high=past_high, vocab=vocab)


def _named(name, **case):
    return case if name is None else {"name": name, **case}


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "chunk", "norm", "norm", "logits", "logits", "history"])
    if kind == "chunk":
        heads = rng.choice([8, 16, 20, 32, 64, 128])
        batch = _log(rng, 1, 16)
        count = _log(rng, 1, max(1, min(4096, 262144 // (heads * batch))))
        # At most the rows and products of the largest listed case.
        top = max(1, min(61440, 65536 // batch, 4_000_000_000 // (batch * count * heads) - count))
        ctx = _log(rng, 1, top)
        return _chunk(None, batch=batch, heads=heads, count_low=rng.choice([1, count]), count_high=count,
                      ctx_low=rng.choice([0, ctx]), ctx_high=ctx)
    if kind == "norm":
        index = rng.random() < 0.5
        dim = 128 if index else rng.choice([64, 128, 192, 256, 512])
        rotary = rng.choice([32, 64, 128, dim]) if dim >= 128 else rng.choice([32, 64])
        heads, keys = rng.choice([1, 8, 20, 32, 64]), 1 if index else rng.choice([1, 4, 8])
        norms = [None, "rms", "layer"]
        return _norm(None, tokens=_log(rng, 1, 8192 * 65 * 128 // (2 * (heads + keys) * dim)), heads=heads, keys=keys, dim=dim,
                     rotary=rotary, layout=rng.choice(["interleaved", "half"]), scaling=rng.choice(["none", "linear", "yarn"]),
                     query_norm=rng.choice(norms), key_norm=rng.choice(norms), index=index,
                     dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), top=_log(rng, 100, 1 << 20))
    vocab = _log(rng, 500, 131072)
    past = _log(rng, 1, 16384)
    if kind == "history":
        return _history(None, batch=_log(rng, 1, 32), past_low=rng.randint(0, past), past_high=past, vocab=vocab)
    high = _log(rng, 1, 33)
    return _logits(None, batch=_log(rng, 1, max(1, min(64, 40_000_000 // (vocab * high)))), rows_low=rng.randint(1, high),
                   rows_high=high, vocab=vocab, past_low=rng.randint(0, past), past_high=past,
                   biases=rng.choice([0, rng.randint(1, 200)]), masked=rng.random() < 0.4,
                   dtype=rng.choice(["fp32", "bf16", "fp16"]))


# --- inputs -------------------------------------------------------------------------------


def prepare(case, seed):
    return {"chunk": _prepare_chunk, "norm": _prepare_norm, "logits": _prepare_logits,
            "history": _prepare_history}[case["kind"]](case, seed)


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE)


def _device(values, dtype):
    return torch.from_numpy(np.ascontiguousarray(values)).to(dtype).to(DEVICE)


def _spread(low, high, count):
    """Whole numbers between low and high, the first of them high, spread evenly in no order."""
    return np.asarray([high - int((i * 0.6180339887498949 % 1.0) * (high - low + 1)) for i in range(count)], np.int64)


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)])


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


def _chunk_lengths(case):
    """(tokens of every chunk, cached rows before them)."""
    counts = _spread(case["count_low"], case["count_high"], case["batch"])
    return counts, _spread(case["ctx_low"], case["ctx_high"], case["batch"])[::-1].copy()


def _prepare_chunk(case, seed):
    gen, rng = _generator(seed), np.random.default_rng(seed)
    batch, heads = case["batch"], case["heads"]
    counts, past = _chunk_lengths(case)
    lens = counts + past
    blocks = -(-lens // BLOCK)
    pages = int(blocks.sum())
    kv = _kv_rows(gen, pages * BLOCK).view(pages, BLOCK, ROW_BYTES)
    table, at, order = np.full((batch, int(blocks.max())), -1, np.int32), 0, rng.permutation(pages)
    for b, n in enumerate(blocks):
        table[b, :n] = order[at:at + n]
        at += n
    tokens = int(counts.sum())
    state = {"kind": "chunk", "kv": kv, "table": _device(table, torch.int32), "lens": _device(lens, torch.int32),
             "starts": _device(_starts(counts), torch.int32), "counts": counts.tolist(), "rows": lens.tolist(),
             "query": _normal(gen, tokens, heads, KEY_DIM).to(torch.bfloat16)}
    if own:
        import kvip_amd

        op = kvip_amd.ChunkAttention(torch, batch=batch, heads=heads, max_tokens=tokens, max_context=int(lens.max()),
                                     max_rows=pages * BLOCK, device=DEVICE)
        state["op"] = op.bind(state["query"], kv, state["table"], state["lens"], state["starts"])
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


def _prepare_norm(case, seed):
    gen, dtype = _generator(seed), _DTYPES[case["dtype"]]
    tokens, heads, keys, dim, index = case["tokens"], case["heads"], case["keys"], case["dim"], case["index"]
    frequencies, factor = _frequencies(case["rotary"], _SCALINGS[case["scaling"]])
    # Queries and keys are slices of what one projection wrote, keys with an offset that a norm takes out.
    projected = _normal(gen, tokens, (heads + keys) * dim)
    projected[:, heads * dim:] = projected[:, heads * dim:] * 1.7 + 0.4
    projected = projected.to(dtype)
    state = {"kind": "norm", "index": index, "query": projected[:, :heads * dim].view(tokens, heads, dim),
             "key": projected[:, heads * dim:].view(tokens, keys, dim),
             "positions": torch.randint(0, case["top"], (tokens,), generator=gen, device=DEVICE),
             "frequencies": torch.tensor(frequencies, dtype=torch.float64, device=DEVICE), "factor": factor,
             "half": case["layout"] == "half", "rotary": case["rotary"]}
    for x, norm in (("query", case["query_norm"]), ("key", case["key_norm"])):
        state[x + "_norm"] = None if norm == "none" else norm
        state[x + "_weight"] = None if norm == "none" else 1.0 + 0.2 * _normal(gen, dim)
        state[x + "_bias"] = 0.1 * _normal(gen, dim) if norm == "layer" else None
    if index:
        pages = 2 * -(-tokens // BLOCK)
        state.update(pages=torch.zeros((pages, BLOCK, INDEX_DIM), dtype=torch.float8_e4m3fn, device=DEVICE),
                     scales=torch.ones((pages, BLOCK), device=DEVICE),
                     slots=torch.randperm(pages * BLOCK, generator=gen, device=DEVICE)[:tokens].contiguous())
        state["slots"][tokens // 2::97] = -1  # padded tokens
    if own:
        import kvip_amd

        scaling = _SCALINGS[case["scaling"]]
        rotary = kvip_amd.Rotary(torch, rotary_dim=case["rotary"], layout=case["layout"],
                                 scaling=None if scaling["kind"] == "none" else scaling, device=DEVICE)
        op = kvip_amd.NormRotary(torch, rotary=rotary, dim=dim, query_norm=state["query_norm"], key_norm=state["key_norm"],
                                 epsilon=EPSILON)
        weights = {x: state[x] for x in ("query_weight", "query_bias", "key_weight", "key_bias")}
        state["query_out"] = torch.empty((tokens, heads, dim), dtype=torch.float8_e4m3fn if index else dtype, device=DEVICE)
        if index:
            state["query_scale"] = torch.empty((tokens, heads), device=DEVICE)
            op.bind(state["positions"], state["query"], state["key"], query_out=state["query_out"],
                    query_scale=state["query_scale"], slots=state["slots"], key_cache=state["pages"],
                    key_scales=state["scales"], **weights)
        else:
            state["key_out"] = torch.empty((tokens, keys, dim), dtype=dtype, device=DEVICE)
            op.bind(state["positions"], state["query"], state["key"], query_out=state["query_out"],
                    key_out=state["key_out"], **weights)
        state["op"] = op
    return state


def _tokens(rng, count, vocab):
    """Tokens as texts have them: a few often, most seldom."""
    return np.minimum((vocab * rng.random(count) ** 4).astype(np.int64) * 7919 % vocab, vocab - 1)


def _histories(case, rng):
    """(packed tokens, how many each request has, how many of these are its prompt's)."""
    counts = _spread(case["past_low"], case["past_high"], case["batch"])
    return _tokens(rng, int(counts.sum()), case["vocab"]), counts, counts * 3 // 4


def _prepare_history(case, seed):
    rng = np.random.default_rng(seed)
    tokens, counts, prompts = _histories(case, rng)
    batch = case["batch"]
    state = {"kind": "history", "vocab": case["vocab"], "batch": batch, "tokens": _device(tokens, torch.int64),
             "starts": _device(_starts(counts), torch.int32), "prompts": _device(prompts, torch.int32),
             "requests": _device(rng.permutation(batch), torch.int32)}
    if own:
        import kvip_amd

        state["op"] = kvip_amd.TokenHistory(torch, batch=batch, vocab=case["vocab"], device=DEVICE)
    return state


def _trees(rng, counts):
    """Parents (within the request, -1 for the root) of every step token."""
    parents = []
    for n in counts:
        parents += [-1 if i == 0 else int(rng.integers(max(0, i - 4), i)) for i in range(n)]
    return np.asarray(parents, np.int32)


def _seen(parents, counts):
    """Visibility bits of every step token: itself and its ancestors, as its request's tokens."""
    bits, at = np.zeros(len(parents), np.uint64), 0
    for n in counts:
        for i in range(n):
            own_bit, up = np.uint64(1) << np.uint64(i), parents[at + i]
            bits[at + i] = own_bit | (bits[at + up] if up >= 0 else np.uint64(0))
        at += n
    return bits.view(np.int64)


def _words(vocab):
    return -(-vocab // 32)


def _prepare_logits(case, seed):
    gen, rng = _generator(seed), np.random.default_rng(seed)
    batch, vocab = case["batch"], case["vocab"]
    counts = _spread(case["rows_low"], case["rows_high"], batch)
    rows, starts = int(counts.sum()), _starts(counts)
    past, past_counts, prompts = _histories(case, rng)

    def per_request(low, high):
        return _device(rng.uniform(low, high, batch), torch.float32)

    temperature = per_request(0.5, 1.3)
    temperature[3::8] = 0.0  # some requests take the largest
    state = {"kind": "logits", "batch": batch, "vocab": vocab,
             "logits": (4.0 * _normal(gen, rows, vocab)).to(_DTYPES[case["dtype"]]),
             "starts": _device(starts, torch.int32), "tokens": _device(_tokens(rng, rows, vocab), torch.int64),
             "seen": _device(_seen(_trees(rng, counts), counts), torch.int64), "nodes": int(counts.max()),
             "temperature": temperature, "repetition": per_request(1.02, 1.4), "presence": per_request(0.0, 0.8),
             "frequency": per_request(0.0, 0.3), "allowed": None, "bias_tokens": None, "bias_values": None,
             "past": _device(past, torch.int64), "past_starts": _device(_starts(past_counts), torch.int32),
             "prompts": _device(prompts, torch.int32)}
    if case["biases"]:
        n = min(case["biases"], vocab)
        tokens = np.stack([rng.permutation(vocab)[:n] for _ in range(batch)])
        tokens[1::3, n // 2:] = -1  # requests with fewer
        state.update(bias_tokens=_device(tokens, torch.int32), bias_values=_device(rng.uniform(-6, 6, (batch, n)), torch.float32))
    if case["masked"]:
        # Grammars allow a few tokens of the vocabulary or most of them.
        words = torch.randint(-2 ** 31, 2 ** 31, (rows, _words(vocab)), generator=gen, device=DEVICE)
        some = torch.randint(-2 ** 31, 2 ** 31, (rows, _words(vocab)), generator=gen, device=DEVICE)
        state["allowed"] = torch.where((torch.arange(rows, device=DEVICE) % 2 == 0)[:, None], words & some & (some >> 3),
                                       words | some).int()
    if own:
        import kvip_amd

        history = kvip_amd.TokenHistory(torch, batch=batch, vocab=vocab, device=DEVICE)
        history.load(torch.arange(batch, dtype=torch.int32, device=DEVICE), state["past"], state["past_starts"], state["prompts"])
        op = kvip_amd.LogitProcessor(torch, batch=batch, max_tokens=rows, vocab=vocab, device=DEVICE)
        state["op"] = op.bind(state["logits"], state["starts"], temperature=temperature, history=history,
                              repetition=state["repetition"], presence=state["presence"], frequency=state["frequency"],
                              tokens=state["tokens"], visible=state["seen"], bias_tokens=state["bias_tokens"],
                              bias_values=state["bias_values"], allowed=state["allowed"])
    else:
        order = torch.arange(batch, device=DEVICE)
        state["held"] = _counted(state["past"], state["past_starts"], state["prompts"], order, vocab)
    return state


# --- one pass -----------------------------------------------------------------------------


def run(state):
    if own:
        return {"chunk": _own_chunk, "norm": _own_norm, "logits": _own_logits, "history": _own_history}[state["kind"]](state)
    return {"chunk": _plain_chunk, "norm": _plain_norm, "logits": _plain_logits, "history": _plain_history}[state["kind"]](state)


def _own_chunk(state):
    return [state["op"]()]


def _own_norm(state):
    state["op"]()
    if state["index"]:
        return [state["query_out"], state["query_scale"], state["pages"], state["scales"]]
    return [state["query_out"], state["key_out"]]


def _own_logits(state):
    return [state["op"]()]


def _own_history(state):
    op = state["op"]
    op.load(state["requests"], state["tokens"], state["starts"], state["prompts"])
    return [op.counts, op.seen]


# --- the plain forms ----------------------------------------------------------------------


def _plain_chunk(s):
    """softmax(scale * q k) v in 32 bits over every cached row up to the token's own, request by request."""
    heads, out, at = s["query"].shape[1], [], 0
    for b, (n, length) in enumerate(zip(s["counts"], s["rows"])):
        rows = s["kv"][s["table"][b, :-(-length // BLOCK)].long()].view(-1, ROW_BYTES)[:length]
        scales = rows[:, 640:656].contiguous().view(torch.float32)
        value = (rows[:, :512].contiguous().view(torch.float8_e4m3fn).float().view(length, 4, 128) * scales[..., None]).view(length, -1)
        key = torch.cat([value, rows[:, 512:640].contiguous().view(torch.bfloat16).float()], -1).t().contiguous()
        place = torch.arange(length, device=DEVICE)
        step = max(1, (1 << 28) // (heads * length))
        for first in range(0, n, step):
            query = s["query"][at + first:at + min(first + step, n)].float()
            last = torch.arange(length - n + first, length - n + first + len(query), device=DEVICE)
            logits = (query.view(-1, KEY_DIM) @ key).view(len(query), heads, length) * KEY_DIM ** -0.5
            logits = logits.masked_fill((place > last[:, None])[:, None, :], float("-inf"))
            weight = torch.exp(logits - logits.amax(-1, keepdim=True))
            weight = (weight / weight.sum(-1, keepdim=True)).view(-1, length)
            out.append((weight @ value).view(len(query), heads, VALUE_DIM).to(torch.bfloat16))
        at += n
    return [torch.cat(out)]


def _normed(x, norm, weight, bias):
    if norm is None:
        return x
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPSILON) * weight
    return x if bias is None else x + bias


def _turned(x, s):
    """x fp32 [tokens, heads, dim] with its first features turned by the tokens' angles."""
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = ((f(angle) * s["factor"]).float()[:, None] for f in (torch.cos, torch.sin))
    part = x[..., :s["rotary"]]
    if s["half"]:
        a, b = part.chunk(2, -1)
        part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([part, x[..., s["rotary"]:]], -1)


def _quantised(x):
    """fp8 values and the scale per head that they are multiplied by."""
    largest = x.abs().amax(-1)
    scale = torch.where(largest > 0, largest / 448, torch.ones_like(largest))
    return (x / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _plain_norm(s):
    query = _turned(_normed(s["query"].float(), s["query_norm"], s["query_weight"], s["query_bias"]), s)
    key = _turned(_normed(s["key"].float(), s["key_norm"], s["key_weight"], s["key_bias"]), s)
    if not s["index"]:
        return [query.to(s["query"].dtype), key.to(s["key"].dtype)]
    kept = s["slots"] >= 0
    values, scales = _quantised(key[:, 0])
    at = s["slots"][kept]
    s["pages"].view(torch.uint8).view(-1, INDEX_DIM)[at] = values.view(torch.uint8)[kept]
    s["scales"].view(-1)[at] = scales[kept]
    return [*_quantised(query), s["pages"], s["scales"]]


def _counted(tokens, starts, prompts, requests, vocab):
    """(how often each request wrote each token, whether it holds it at all)."""
    place = torch.arange(len(tokens), device=DEVICE)
    owner = torch.searchsorted(starts[1:].long(), place, right=True)
    prompt = place - starts[owner].long() < prompts[owner].long()
    at = requests[owner].long() * vocab + tokens
    counts = torch.zeros(len(requests) * vocab, dtype=torch.int32, device=DEVICE)
    counts.index_add_(0, at, (~prompt).int())
    held = torch.zeros(len(requests) * vocab, dtype=torch.bool, device=DEVICE)
    held[at] = True
    return counts.view(-1, vocab), held.view(-1, vocab)


def _packed(bits):
    """bool [n, vocab] as int32 words, bit v % 32 of word v / 32."""
    n, vocab = bits.shape
    whole = torch.zeros((n, _words(vocab) * 32), dtype=torch.int64, device=DEVICE)
    whole[:, :vocab] = bits
    words = (whole.view(n, -1, 32) << torch.arange(32, device=DEVICE)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()


def _plain_history(s):
    counts, held = _counted(s["tokens"], s["starts"], s["prompts"], s["requests"], s["vocab"])
    return [counts, _packed(held)]


def _plain_logits(s):
    vocab, starts = s["vocab"], s["starts"].long()
    rows = torch.arange(len(s["logits"]), device=DEVICE)
    owner = torch.searchsorted(starts[1:], rows, right=True)
    counts, held = s["held"][0][owner], s["held"][1][owner]
    # Drafted tokens on the way to a row count as written; a request's token 0 is in its history already.
    node = torch.arange(1, max(s["nodes"], 2), device=DEVICE)
    at = starts[owner][:, None] + node
    there = (at < starts[owner + 1][:, None]) & ((s["seen"][:, None] >> node) & 1 == 1)
    drafted = s["tokens"][at.clamp(max=len(rows) - 1)]
    counts = counts.scatter_add(1, drafted, there.int())
    held = held | (counts > 0)
    x = s["logits"].float()
    repetition = s["repetition"][owner][:, None]
    x = torch.where(held, torch.where(x > 0, x / repetition, x * repetition), x)
    x = x - torch.where(counts > 0, s["presence"][owner][:, None] + s["frequency"][owner][:, None] * counts, torch.zeros_like(x))
    if s["bias_tokens"] is not None:
        names, values = s["bias_tokens"][owner].long(), s["bias_values"][owner]
        x = x.scatter_add(1, names.clamp(min=0), torch.where(names >= 0, values, torch.zeros_like(values)))
    if s["allowed"] is not None:
        v = torch.arange(vocab, device=DEVICE)
        x = x.masked_fill((s["allowed"][:, v // 32] >> (v % 32)) & 1 == 0, float("-inf"))
    temperature = s["temperature"][owner][:, None]
    largest = x.amax(1, keepdim=True)
    weight = torch.exp((x - largest) / torch.where(temperature > 0, temperature, torch.ones_like(temperature)))
    first = torch.where(x == largest, torch.arange(vocab, device=DEVICE), vocab).amin(1, keepdim=True)
    weight = torch.where(temperature > 0, weight, (torch.arange(vocab, device=DEVICE) == first).float())
    return [weight / weight.sum(1, keepdim=True)]


# --- the operators in 64 bits -------------------------------------------------------------


def exact(case, seed):
    if case["kind"] == "history":
        return None  # whole numbers
    state = prepare(case, seed)
    return {"chunk": _exact_chunk, "norm": _exact_norm, "logits": _exact_logits}[case["kind"]](state)


def _exact_chunk(s):
    heads, starts = s["query"].shape[1], s["starts"].tolist()
    out = torch.empty((starts[-1], heads, VALUE_DIM), dtype=torch.float64, device=DEVICE)
    for b, length in enumerate(s["lens"].tolist()):
        rows = s["kv"][s["table"][b, :-(-length // BLOCK)].long()].reshape(-1, ROW_BYTES)[:length].contiguous()
        scale = rows[:, 640:656].contiguous().view(torch.float32).double().repeat_interleave(128, 1)
        value = rows[:, :512].contiguous().view(torch.float8_e4m3fn).double() * scale
        key = torch.cat([value, rows[:, 512:640].contiguous().view(torch.bfloat16).double()], 1).t().contiguous()
        tokens = starts[b + 1] - starts[b]
        step = max(1, (1 << 27) // (heads * length))
        for first in range(0, tokens, step):
            here = slice(starts[b] + first, starts[b] + min(first + step, tokens))
            reach = length - tokens + min(first + step, tokens)  # rows that the last of these tokens sees
            logits = s["query"][here].double().flatten(0, 1) @ key[:, :reach].contiguous() / math.sqrt(KEY_DIM)
            logits = logits.view(-1, heads, reach)
            hidden = torch.ones((len(logits), reach), dtype=torch.bool, device=DEVICE).triu(length - tokens + first + 1)
            weight = torch.softmax(logits.masked_fill_(hidden[:, None], -math.inf), -1).view(-1, reach)
            out[here] = (weight @ value[:reach]).view(-1, heads, VALUE_DIM)
    return [out]


def _exact_heads(x, kind, weight, bias, s):
    """A head's features normed, then each pair as a complex number times e^(i angle)."""
    y = x.double()
    if kind is not None:
        if kind == "layer":
            variance, mean = torch.var_mean(y, -1, correction=0, keepdim=True)
            y = (y - mean) * torch.rsqrt(variance + EPSILON)
        else:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPSILON)
        y = y * weight.double()
        y = y if bias is None else y + bias.double()
    r = s["rotary"]
    angle = torch.outer(s["positions"].double(), s["frequencies"])
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)[:, None]
    y = y.clone()
    if s["half"]:
        pairs = torch.complex(y[..., :r // 2].contiguous(), y[..., r // 2:r].contiguous()) * turn
        y[..., :r // 2], y[..., r // 2:r] = pairs.real, pairs.imag
    else:
        pairs = torch.complex(y[..., 0:r:2].contiguous(), y[..., 1:r:2].contiguous()) * turn
        y[..., 0:r:2], y[..., 1:r:2] = pairs.real, pairs.imag
    return y


def _exact_codes(y):
    """e4m3: steps of 2^(exponent - 3), the exponent at least -6; halves to the even step."""
    scale = y.abs().amax(-1) / 448
    scale[scale == 0] = 1.0
    y = y / scale[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
    return torch.round(y / step) * step, scale


def _exact_norm(s):
    query = _exact_heads(s["query"], s["query_norm"], s["query_weight"], s["query_bias"], s)
    key = _exact_heads(s["key"], s["key_norm"], s["key_weight"], s["key_bias"], s)
    if not s["index"]:
        return [query, key]
    pages, scales = s["pages"].double().view(-1, INDEX_DIM), s["scales"].double().view(-1)
    kept = s["slots"] >= 0
    codes, per_key = _exact_codes(key[:, 0])
    pages[s["slots"][kept]], scales[s["slots"][kept]] = codes[kept], per_key[kept]
    return [*_exact_codes(query), pages.view(s["pages"].shape), scales.view(s["scales"].shape)]


def _exact_logits(s):
    vocab, starts, past = s["vocab"], s["starts"].tolist(), s["past_starts"].tolist()
    out = torch.empty((starts[-1], vocab), dtype=torch.float64, device=DEVICE)
    numbers = {x: s[x].double().tolist() for x in ("temperature", "repetition", "presence", "frequency")}
    tokens, seen = s["tokens"].tolist(), s["seen"].tolist()
    for b in range(s["batch"]):
        history = s["past"][past[b]:past[b + 1]]
        prompt = int(s["prompts"][b])
        for row in range(starts[b], starts[b + 1]):
            way = [tokens[starts[b] + i] for i in range(1, starts[b + 1] - starts[b]) if seen[row] >> i & 1]
            way = torch.tensor(way, dtype=torch.int64, device=DEVICE)
            written = torch.bincount(torch.cat([history[prompt:], way]), minlength=vocab).double()
            held = (torch.bincount(torch.cat([history, way]), minlength=vocab) > 0).double()
            x = s["logits"][row].double()
            x = x * (1 - held) + held * torch.where(x > 0, x / numbers["repetition"][b], x * numbers["repetition"][b])
            x = x - numbers["frequency"][b] * written - numbers["presence"][b] * (written > 0).double()
            if s["bias_tokens"] is not None:
                named = s["bias_tokens"][b] >= 0
                x.index_add_(0, s["bias_tokens"][b][named].long(), s["bias_values"][b][named].double())
            if s["allowed"] is not None:
                bits = (s["allowed"][row][:, None] >> torch.arange(32, device=DEVICE)) & 1
                x[bits.view(-1)[:vocab] == 0] = -math.inf
            if numbers["temperature"][b] > 0:
                out[row] = torch.softmax(x / numbers["temperature"][b], 0)
            else:
                out[row] = 0.0
                out[row, int(torch.nonzero(x == x.max())[0])] = 1.0
    return [out]


# --- what a pass cannot do without --------------------------------------------------------


def work(case):
    """Bytes of every input read once and every output written once, and the operations."""
    kind, batch = case["kind"], case.get("batch")
    if kind == "chunk":
        counts, past = _chunk_lengths(case)
        rows = float(counts.sum()) * case["heads"]
        pairs = float((counts * past + counts * (counts + 1) // 2).sum()) * case["heads"]  # (query, row) that it sees
        return {"bytes": float((counts + past).sum()) * (ROW_BYTES + 4 / BLOCK) + rows * (KEY_DIM + VALUE_DIM) * 2 + 12 * batch,
                "flops": 2.0 * (KEY_DIM + VALUE_DIM) * pairs}
    if kind == "norm":
        tokens, values = case["tokens"], case["tokens"] * (case["heads"] + case["keys"]) * case["dim"]
        width = 4 if case["dtype"] == "fp32" else 2
        if case["index"]:
            return {"bytes": values * (width + 1.0) + tokens * (16 + 4.0 * (case["heads"] + 1)), "flops": 8.0 * values}
        return {"bytes": 2.0 * values * width + 8 * tokens, "flops": 8.0 * values}
    if kind == "history":
        past = int(_spread(case["past_low"], case["past_high"], batch).sum())
        return {"bytes": 8.0 * past + batch * (4.0 * case["vocab"] + 4.0 * _words(case["vocab"]) + 12), "flops": float(past)}
    rows = int(_spread(case["rows_low"], case["rows_high"], batch).sum())
    past = int(_spread(case["past_low"], case["past_high"], batch).sum())
    width, words = 4 if case["dtype"] == "fp32" else 2, 4.0 * _words(case["vocab"])
    # Probabilities are written in 32 bits; a request's penalties need its tokens' bits and the counts of those it holds.
    return {"bytes": rows * (case["vocab"] * (width + 4.0) + 16 + (words if case["masked"] else 0)) + batch * (words + 16) +
            4.0 * past + 8.0 * case["biases"] * batch, "flops": 8.0 * rows * case["vocab"]}
