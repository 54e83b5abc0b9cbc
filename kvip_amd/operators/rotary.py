"""Rotary positions and the rows of the paged KV cache: `kvip_amd.Rotary`, `kvip_amd.KvRowStore`.

`Rotary` turns the first `rotary_dim` features of every head of queries and keys by their tokens'
positions: interleaved pairs (2 i, 2 i + 1) or halves (i, rotary_dim / 2 + i), whole heads or a part, on
strided views, in place or into another array (a projection's rotary part into the query that
`kvip_amd.TreeAttention` and `kvip_amd.SparseAttention` read), with frequencies scaled for long contexts. `KvRowStore` writes
tokens into the paged cache that those read: latents quantised to fp8 with one scale per 128 features,
rotary features turned on the way. Both bind their tensors once and then only enqueue (capturable).
`include/kvip_hip_draft.h` states the arithmetic. The reference leaves these steps to its engine.
"""
from __future__ import annotations

import math

from kvip_amd.runtime import abi

BLOCK_TOKENS = 128
LATENT_DIM = 512
ROPE_DIM = 64
ROW_BYTES = 656


def _dtype_code(torch, dtype, what):
    codes = {torch.bfloat16: abi.DTYPE_BF16, torch.float16: abi.DTYPE_FP16, torch.float32: abi.DTYPE_FP32}
    abi.require(dtype in codes, f"{what} must be bfloat16, float16 or float32")
    return codes[dtype]


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None):
    """([angle per position of each pair], magnitude) in 64 bits: base^(-2 i / rotary_dim), and by `scaling`
      {"kind": "linear", "factor": s}    every frequency divided by s (positions interpolated);
      {"kind": "ntk", "factor": s}       base * s^(rotary_dim / (rotary_dim - 2)) instead of base;
      {"kind": "yarn", "factor": s, "original": context, "beta_fast": 32, "beta_slow": 1}
          pairs that turn more than beta_fast times over the original context keep their frequency, those
          below beta_slow are divided by s, linearly in between (Peng et al. 2023); magnitude
          0.1 ln(s) + 1 unless "magnitude" is given."""
    abi.require(rotary_dim % 2 == 0 and 2 <= rotary_dim <= 512, "rotary_dim must be even, in 2..512")
    abi.require(math.isfinite(base) and base > 1.0, "base must be above 1")
    scaling = dict(scaling or {"kind": "none"})
    kind = scaling.pop("kind", None)
    allowed = {"none": (), "linear": ("factor",), "ntk": ("factor",),
               "yarn": ("factor", "original", "beta_fast", "beta_slow", "magnitude")}
    abi.require(kind in allowed, "scaling kind must be none, linear, ntk or yarn")
    abi.require(set(scaling) <= set(allowed[kind]), f"{kind} scaling takes {', '.join(allowed[kind]) or 'nothing'}")
    pairs = rotary_dim // 2
    if kind == "none":
        return [base ** (-2.0 * i / rotary_dim) for i in range(pairs)], 1.0
    abi.require("factor" in scaling and math.isfinite(scaling["factor"]) and scaling["factor"] >= 1.0,
                "scaling needs a factor of at least 1")
    factor = float(scaling["factor"])
    if kind == "linear":
        return [base ** (-2.0 * i / rotary_dim) / factor for i in range(pairs)], 1.0
    if kind == "ntk":
        abi.require(rotary_dim > 2, "ntk scaling needs a rotary_dim above 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
        return [base ** (-2.0 * i / rotary_dim) for i in range(pairs)], 1.0
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
    abi.require(scaling.get("original", 0) >= 1 and fast > slow > 0, "yarn scaling needs original >= 1, beta_fast > beta_slow > 0")

    def pair_turning(turns):
        return rotary_dim * math.log(scaling["original"] / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    low = max(math.floor(pair_turning(fast)), 0)
    high = min(math.ceil(pair_turning(slow)), rotary_dim - 1)
    out = []
    for i in range(pairs):
        f = base ** (-2.0 * i / rotary_dim)
        stretched = min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0)
        out.append(f * (1.0 - stretched) + f / factor * stretched)
    return out, float(scaling.get("magnitude", 0.1 * math.log(factor) + 1.0))


class Rotary:
    """layout "interleaved" or "half"; base and scaling as `rotary_frequencies`. `bind` validates a call's
    tensors, `__call__` enqueues it on the current stream."""

    def __init__(self, torch, *, rotary_dim, device, layout="interleaved", base=10000.0, scaling=None):
        abi.require(layout in ("interleaved", "half"), "layout must be interleaved or half")
        values, self.magnitude = rotary_frequencies(rotary_dim, base, scaling)
        self.torch, self.device = torch, abi.device_of(torch, device)
        abi.require(self.device.type == "cuda", "rotary positions run on the GPU (kvip_amd has no CPU path)")
        self.rotary_dim, self.half = int(rotary_dim), layout == "half"
        self.frequencies = torch.tensor(values, dtype=torch.float64, device=self.device)
        self.library = abi.load_library()
        self.args = None

    def _tensor(self, x, out, tokens, what):
        """(struct, heads view) of one array and its output, [tokens, heads, dim] or [tokens, dim]."""
        for t in (x, out):
            abi.require(t.dim() in (2, 3) and t.shape[0] == tokens and t.shape[-1] >= self.rotary_dim,
                        f"{what} must be [{tokens}, heads, dim] or [{tokens}, dim] with dim >= {self.rotary_dim}")
            abi.require(t.stride(-1) == 1, f"{what}: the last dimension must be contiguous")
            abi.require(t.device == self.device, f"{what} must be on {self.device}")
        abi.require(x.shape == out.shape and x.dtype == out.dtype, f"{what} and its output must have one shape and type")
        heads = int(x.shape[1]) if x.dim() == 3 else 1
        strides = [(t.stride(0), t.stride(1) if t.dim() == 3 else 0) for t in (x, out)]
        abi.require(1 <= heads <= 65536 and x.shape[-1] <= 65536, f"{what} must have 1..65536 heads and features")
        same = x.data_ptr() == out.data_ptr()
        abi.require(not same or strides[0] == strides[1], f"{what}: an array turned in place keeps its strides")
        (by_token, by_head), dim = strides[1], int(x.shape[-1])
        apart = (heads <= 1 or by_head >= dim) and (tokens <= 1 or by_token >= dim) and (
            tokens <= 1 or heads <= 1 or by_token >= by_head * (heads - 1) + dim or by_head >= by_token * (tokens - 1) + dim)
        abi.require(apart, f"{what}: output rows must not overlap")
        return abi.RotaryTensor(x=x.data_ptr(), out=out.data_ptr(), x_token=strides[0][0], x_head=strides[0][1],
                                out_token=strides[1][0], out_head=strides[1][1], heads=heads, dim=int(x.shape[-1]))

    def bind(self, positions, query, key=None, *, query_out=None, key_out=None, inverse=False):
        """positions int64 [tokens]; query (and key) [tokens, heads, dim] or [tokens, dim] of one type (bf16,
        fp16, fp32), dim >= rotary_dim, strided as long as the last dimension is contiguous. Without an
        output the array is turned in place; with one, features behind rotary_dim are copied. An output
        does not overlap another array. inverse: turned by the negative angle, times the same magnitude: the gradient
        of a turn, and what undoes it where the magnitude is 1 (else up to the magnitude's square)."""
        t = self.torch
        abi.require(positions.dtype == t.int64 and positions.dim() == 1 and positions.is_contiguous() and
                    positions.device == self.device, f"positions must be contiguous int64 [tokens] on {self.device}")
        tokens = int(positions.shape[0])
        query_out = query if query_out is None else query_out
        abi.require(key is not None or key_out is None, "key_out needs a key")
        key_out = key if key_out is None else key_out
        code = _dtype_code(t, query.dtype, "query")
        abi.require(key is None or key.dtype == query.dtype, "key must have the query's type")
        args = abi.RotaryArgs(positions=abi.ptr(positions), frequencies=abi.ptr(self.frequencies), tokens=tokens,
                              rotary_dim=self.rotary_dim, half=int(self.half), inverse=int(bool(inverse)), dtype=code,
                              magnitude=self.magnitude)
        args.tensors[0] = self._tensor(query, query_out, tokens, "query")
        if key is not None:
            args.tensors[1] = self._tensor(key, key_out, tokens, "key")
        self.args, self._outputs = args, (query_out, key_out)
        self._bound = (positions, query, key, query_out, key_out)
        return self

    def __call__(self):
        """Returns (query output, key output or None)."""
        abi.require(self.args is not None, "bind() the rotary tensors first")
        if self.args.tokens:
            abi.launch(self.torch, self.device, self.library.kvip_hip_rotary, self.args, "rotary positions")
        return self._outputs


class KvRowStore:
    """Writes tokens' rows into a paged cache: kv_cache uint8 (or float8_e4m3fn) [blocks, 128, row_stride] or
    [blocks, 128, 1, row_stride] with rows of 656 bytes, as `kvip_amd.SparseAttention` reads it. rotary: a
    `Rotary` of 64 features turns the rotary features by the tokens' positions (None: they come turned)."""

    def __init__(self, torch, *, kv_cache, rotary=None):
        if kv_cache.dim() == 4:
            abi.require(kv_cache.shape[2] == 1, "kv_cache must be [blocks, 128, 1, row_stride]")
            kv_cache = kv_cache[:, :, 0]
        abi.require(kv_cache.dtype in (torch.uint8, torch.float8_e4m3fn) and kv_cache.dim() == 3 and
                    kv_cache.shape[1] == BLOCK_TOKENS and kv_cache.shape[2] >= ROW_BYTES and kv_cache.stride(2) == 1,
                    "kv_cache must be 1-byte [blocks, 128, row_stride >= 656] with contiguous rows")
        abi.require(kv_cache.device.type == "cuda", "row stores run on the GPU (kvip_amd has no CPU path)")
        self.torch, self.device, self.kv_cache, self.rotary = torch, kv_cache.device, kv_cache, rotary
        abi.require(rotary is None or (rotary.rotary_dim == ROPE_DIM and rotary.device == self.device),
                    "rotary must turn 64 features, on the cache's device")
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.library = abi.load_library()
        self.args = None

    def bind(self, latent, rope, slots, positions=None):
        """latent [tokens, 512] and rope [tokens, 64] of one type (bf16, fp16, fp32), rows contiguous and at
        any stride; slots int64 [tokens] (page * 128 + row, negative: no row; no slot twice);
        positions int64 [tokens], with a rotary."""
        t = self.torch
        tokens = int(slots.shape[0]) if slots.dim() == 1 else -1
        for x, width, what in ((latent, LATENT_DIM, "latent"), (rope, ROPE_DIM, "rope")):
            abi.require(tuple(x.shape) == (tokens, width) and x.stride(1) == 1 and x.device == self.device,
                        f"{what} must be [tokens, {width}] with contiguous rows on {self.device}")
        abi.require(latent.dtype == rope.dtype, "latent and rope must have one type")
        code = _dtype_code(t, latent.dtype, "latent")
        abi.require((positions is None) == (self.rotary is None), "positions go with a rotary")
        for x in (slots,) if positions is None else (slots, positions):
            abi.require(x.dtype == t.int64 and tuple(x.shape) == (tokens,) and x.is_contiguous() and x.device == self.device,
                        f"slots and positions must be contiguous int64 [tokens] on {self.device}")
        p, kv, rotary = abi.ptr, self.kv_cache, self.rotary
        self.args = abi.RowStoreArgs(
            latent=p(latent), rope=p(rope), slots=p(slots), positions=p(positions),
            frequencies=p(None if rotary is None else rotary.frequencies), kv_cache=p(kv), status=p(self.status),
            latent_stride=latent.stride(0), rope_stride=rope.stride(0), kv_block_stride=kv.stride(0), tokens=tokens,
            row_stride=kv.stride(1), num_blocks=int(kv.shape[0]), half=int(rotary is not None and rotary.half), dtype=code,
            magnitude=1.0 if rotary is None else rotary.magnitude)
        self._bound = (latent, rope, slots, positions)
        return self

    def __call__(self):
        """Enqueues the rows; returns the cache."""
        abi.require(self.args is not None, "bind() the rows first")
        if self.args.tokens:
            abi.launch(self.torch, self.device, self.library.kvip_hip_store_rows, self.args, "row store")
        return self.kv_cache
