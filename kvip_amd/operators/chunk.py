"""Attention of prompt chunks over their requests' paged context: `kvip_amd.ChunkAttention` and
`kvip_amd.chunk_attention`.

The dense counterpart of `kvip_amd.PrefillIndexer` and `kvip_amd.SparseAttention` for chunks of any number of tokens,
for contexts that the selection would take whole and for layers without one: token i of a chunk attends every
cached row of its request up to its own. Rows are the 656-byte rows of the paged KV cache, read through the block
table; requests of a batch may have any lengths and counts (packed rows), decoding ones with a single token among
them. A step of at most 64 tokens per request that are not a chain, or that are few, is `kvip_amd.TreeAttention`'s.
`include/kvip_hip_prompt.h` states the arithmetic. The reference has no counterpart (its attention is its engine's).
"""
from __future__ import annotations

import math

from kvip_amd.runtime import abi

BLOCK_TOKENS = 128
KEY_DIM = 576
VALUE_DIM = 512
ROW_BYTES = 656


class ChunkAttention:
    """Output [max_tokens, heads, 512] (bf16 or fp32), log-sum-exp float32 [max_tokens, heads] (lse=True), status and
    workspace allocated once; `bind` validates a call's tensors, `__call__` enqueues it on the current stream
    (capturable; one object's calls follow one another, as they share its workspace). max_tokens: tokens of a call;
    max_context: cached rows of a request, the chunk's among them; max_rows: cached rows of a call's requests
    together (default batch * max_context), which the workspace holds as fp16, 1152 bytes each, beside 269 MB for the parts
    of contexts that are cut (objects for few rows, up to 64 tokens and 512 * batch of tokens times heads, have neither: up to
    135 MB, and the cache is read as it is). One object serves layer after layer. A request past max_rows gets zeros and sets a
    status bit."""

    def __init__(self, torch, *, batch, heads, max_tokens, max_context, device, max_rows=None, output_dtype=None, lse=False):
        abi.require(1 <= batch <= abi.DRAFT_MAX_BATCH, f"batch must be in 1..{abi.DRAFT_MAX_BATCH}")
        abi.require(1 <= heads <= 128, "chunk attention supports 1..128 heads")
        abi.require(1 <= max_tokens <= abi.DRAFT_MAX_TOKENS, f"max_tokens must be in 1..{abi.DRAFT_MAX_TOKENS}")
        abi.require(1 <= max_context <= 1 << 24, "max_context must be in 1..2^24")
        self.max_blocks = (int(max_context) + BLOCK_TOKENS - 1) // BLOCK_TOKENS
        max_rows = int(batch) * self.max_blocks * BLOCK_TOKENS if max_rows is None else int(max_rows)
        abi.require(1 <= max_rows <= 1 << 31, "max_rows must be in 1..2^31")
        output_dtype = torch.bfloat16 if output_dtype is None else output_dtype
        abi.require(output_dtype in (torch.bfloat16, torch.float32), "the output is bfloat16 or float32")
        self.torch, self.device = torch, abi.device_of(torch, device)
        abi.require(self.device.type == "cuda", "chunk attention runs on the GPU (kvip_amd has no CPU path)")
        self.batch, self.heads, self.max_tokens, self.max_rows = int(batch), int(heads), int(max_tokens), max_rows
        self.library = abi.load_library()
        nbytes = int(self.library.kvip_hip_chunk_attention_workspace_bytes(batch, heads, max_tokens, self.max_blocks, max_rows))
        abi.require(nbytes > 0, "the sizes are too large for one call")
        self.output = torch.zeros((max_tokens, heads, VALUE_DIM), dtype=output_dtype, device=self.device)
        self.lse = torch.zeros((max_tokens, heads), dtype=torch.float32, device=self.device) if lse else None
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self.args = None

    def bind(self, query, kv_cache, block_table, seq_lens, cu_seqlens, scale=KEY_DIM ** -0.5, *, steps=None):
        """query bf16 [max_tokens, heads, 576]; kv_cache 1-byte [blocks, 128, row_stride] (or [blocks, 128, 1,
        row_stride]) with rows of 656 bytes; block_table int32 [batch, blocks of max_context or fewer];
        seq_lens int32 [batch]: cached rows, the chunk's among them; cu_seqlens int32 [batch + 1]. steps int32 [batch]
        (PageTables.steps, read before its commit): requests with 0, which extend refused and which have no rows of
        the step in the cache, get zeros. Rows behind the last token are neither read nor written."""
        t = self.torch
        abi.require(query.dtype == t.bfloat16 and tuple(query.shape) == (self.max_tokens, self.heads, KEY_DIM) and
                    query.is_contiguous(), f"query must be contiguous bfloat16 [{self.max_tokens}, {self.heads}, {KEY_DIM}]")
        if kv_cache.dim() == 4:
            abi.require(kv_cache.shape[2] == 1, "kv_cache must be [blocks, 128, 1, row_stride]")
            kv_cache = kv_cache[:, :, 0]
        abi.require(kv_cache.dtype in (t.uint8, t.float8_e4m3fn) and kv_cache.dim() == 3 and
                    kv_cache.shape[1] == BLOCK_TOKENS and kv_cache.shape[2] >= ROW_BYTES and kv_cache.stride(2) == 1,
                    "kv_cache must be 1-byte [blocks, 128, row_stride >= 656] with contiguous rows")
        abi.require(block_table.dtype == t.int32 and block_table.dim() == 2 and block_table.shape[0] == self.batch and
                    1 <= block_table.shape[1] <= self.max_blocks and block_table.is_contiguous(),
                    f"block_table must be contiguous int32 [{self.batch}, 1..{self.max_blocks}]")
        for x, shape, what in ((seq_lens, (self.batch,), "seq_lens"), (cu_seqlens, (self.batch + 1,), "cu_seqlens"),
                               (steps, (self.batch,), "steps")):
            abi.require(x is None and what == "steps" or
                        (x.dtype == t.int32 and tuple(x.shape) == shape and x.is_contiguous()),
                        f"{what} must be contiguous int32 {list(shape)}")
        for x in (query, kv_cache, block_table, seq_lens, cu_seqlens, steps):
            abi.require(x is None or x.device == self.device, f"chunk attention tensors must be on {self.device}")
        abi.require(math.isfinite(scale), "scale must be finite")
        p = abi.ptr
        self.args = abi.ChunkAttnArgs(
            query=p(query), kv_cache=p(kv_cache), block_table=p(block_table), seq_lens=p(seq_lens), cu_seqlens=p(cu_seqlens),
            steps=p(steps), output=p(self.output), lse=p(self.lse), workspace=p(self.workspace), status=p(self.status),
            kv_block_stride=kv_cache.stride(0), max_rows=self.max_rows, row_stride=kv_cache.stride(1), batch=self.batch,
            heads=self.heads, max_tokens=self.max_tokens, max_blocks=int(block_table.shape[1]),
            num_blocks=int(kv_cache.shape[0]), scale=float(scale),
            output_dtype=abi.DTYPE_FP32 if self.output.dtype == t.float32 else abi.DTYPE_BF16)
        self._bound = (query, kv_cache, block_table, seq_lens, cu_seqlens, steps)
        return self

    def __call__(self):
        abi.require(self.args is not None, "bind() the chunk attention inputs first")
        abi.launch(self.torch, self.device, self.library.kvip_hip_chunk_attention, self.args, "chunk attention")
        return self.output


def chunk_attention(query, kv_cache, block_table, seq_lens, cu_seqlens, scale=KEY_DIM ** -0.5, *, max_rows=None,
                    output_dtype=None, steps=None):
    """One chunk-attention call (arguments as `ChunkAttention`, whose buffers it allocates); returns [rows, heads, 512]. What is
    wrong with tables and lengths, requests past max_rows among it, shows in an object's status alone: without max_rows there is
    room for every request."""
    import torch

    op = ChunkAttention(torch, batch=int(seq_lens.shape[0]), heads=int(query.shape[1]), max_tokens=int(query.shape[0]),
                        max_context=int(block_table.shape[1]) * BLOCK_TOKENS, max_rows=max_rows, device=query.device,
                        output_dtype=output_dtype)
    return op.bind(query, kv_cache, block_table, seq_lens, cu_seqlens, scale, steps=steps)()
