"""Attention of a step's tokens over their requests' whole paged context: `kvip_amd.TreeAttention` and
`kvip_amd.tree_attention`.

The dense counterpart of `kvip_amd.SparseAttention` for steps of drafted tokens: every token of a request
(up to 64, a chain or a tree) attends every cached row of the request and, among the step's own rows,
those that its visibility bits name. Rows are the 656-byte rows of the paged KV cache, read in place through
the block table; requests of a batch may have any lengths and counts (packed rows). `include/kvip_hip_draft.h`
states the arithmetic. The reference has no counterpart (its attention is its engine's).
"""
from __future__ import annotations

import math

from kvip_amd.runtime import abi

BLOCK_TOKENS = 128
KEY_DIM = 576
VALUE_DIM = 512
ROW_BYTES = 656


class TreeAttention:
    """Output [max_tokens, heads, 512] (bf16 or fp32), log-sum-exp float32 [max_tokens, heads] (lse=True) and status
    allocated once; `bind` validates a call's tensors, `__call__` enqueues it on the current stream
    (capturable; one object's calls follow one another, as they share its workspace). max_nodes: step tokens
    of a request (1..64); max_context: its cached rows, the step's among them."""

    def __init__(self, torch, *, batch, heads, max_nodes, max_tokens, max_context, device, output_dtype=None, lse=False):
        abi.require(1 <= batch <= abi.DRAFT_MAX_BATCH, f"batch must be in 1..{abi.DRAFT_MAX_BATCH}")
        abi.require(1 <= heads <= 128, "tree attention supports 1..128 heads")
        abi.require(1 <= max_nodes <= abi.DRAFT_MAX_NODES, f"max_nodes must be in 1..{abi.DRAFT_MAX_NODES}")
        abi.require(1 <= max_tokens <= abi.DRAFT_MAX_TOKENS, f"max_tokens must be in 1..{abi.DRAFT_MAX_TOKENS}")
        abi.require(1 <= max_context <= 1 << 24, "max_context must be in 1..2^24")
        output_dtype = torch.bfloat16 if output_dtype is None else output_dtype
        abi.require(output_dtype in (torch.bfloat16, torch.float32), "the output is bfloat16 or float32")
        self.torch, self.device = torch, abi.device_of(torch, device)
        abi.require(self.device.type == "cuda", "tree attention runs on the GPU (kvip_amd has no CPU path)")
        self.batch, self.heads, self.max_nodes, self.max_tokens = int(batch), int(heads), int(max_nodes), int(max_tokens)
        self.max_blocks = (int(max_context) + BLOCK_TOKENS - 1) // BLOCK_TOKENS
        self.output = torch.zeros((max_tokens, heads, VALUE_DIM), dtype=output_dtype, device=self.device)
        self.lse = torch.zeros((max_tokens, heads), dtype=torch.float32, device=self.device) if lse else None
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.library = abi.load_library()
        # Parts of items that several workgroups share, at most two per workgroup.
        nbytes = int(self.library.kvip_hip_tree_attention_workspace_bytes(batch, heads, max_nodes, self.max_blocks))
        abi.require(nbytes > 0, "batch * heads * max_nodes * max_context is too large for one call")
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self.args = None

    def bind(self, query, kv_cache, block_table, seq_lens, cu_seqlens, visible=None, scale=KEY_DIM ** -0.5, *, steps=None):
        """query bf16 [max_tokens, heads, 576]; kv_cache 1-byte [blocks, 128, row_stride] (or [blocks, 128, 1,
        row_stride]) with rows of 656 bytes; block_table int32 [batch, blocks of max_context or fewer];
        seq_lens int32 [batch]: cached rows, the step's among them; cu_seqlens int32 [batch + 1]; visible int64
        [max_tokens] as kvip_amd.PageTables.extend writes it (None: a chain). steps int32 [batch] (PageTables.steps,
        read before its commit): requests with 0, which extend refused and which have no rows of the step in the
        cache, get zeros. Rows behind the last token are neither read nor written."""
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
        for x, shape, what in ((seq_lens, (self.batch,), "seq_lens"), (cu_seqlens, (self.batch + 1,), "cu_seqlens")):
            abi.require(x.dtype == t.int32 and tuple(x.shape) == shape and x.is_contiguous(),
                        f"{what} must be contiguous int32 {list(shape)}")
        abi.require(visible is None or (visible.dtype == t.int64 and tuple(visible.shape) == (self.max_tokens,) and
                                        visible.is_contiguous()), f"visible must be contiguous int64 [{self.max_tokens}]")
        abi.require(steps is None or (steps.dtype == t.int32 and tuple(steps.shape) == (self.batch,) and steps.is_contiguous()),
                    f"steps must be contiguous int32 [{self.batch}]")
        for x in (query, kv_cache, block_table, seq_lens, cu_seqlens, visible, steps):
            abi.require(x is None or x.device == self.device, f"tree attention tensors must be on {self.device}")
        abi.require(math.isfinite(scale), "scale must be finite")
        p = abi.ptr
        self.args = abi.TreeAttnArgs(
            query=p(query), kv_cache=p(kv_cache), block_table=p(block_table), seq_lens=p(seq_lens), cu_seqlens=p(cu_seqlens),
            visible=p(visible), output=p(self.output), lse=p(self.lse), workspace=p(self.workspace), status=p(self.status),
            kv_block_stride=kv_cache.stride(0), row_stride=kv_cache.stride(1), batch=self.batch, heads=self.heads,
            max_nodes=self.max_nodes, max_tokens=self.max_tokens, max_blocks=int(block_table.shape[1]),
            num_blocks=int(kv_cache.shape[0]), scale=float(scale), steps=p(steps),
            output_dtype=abi.DTYPE_FP32 if self.output.dtype == t.float32 else abi.DTYPE_BF16)
        self._bound = (query, kv_cache, block_table, seq_lens, cu_seqlens, visible, steps)
        return self

    def __call__(self):
        abi.require(self.args is not None, "bind() the tree attention inputs first")
        abi.launch(self.torch, self.device, self.library.kvip_hip_tree_attention, self.args, "tree attention")
        return self.output


def tree_attention(query, kv_cache, block_table, seq_lens, cu_seqlens, visible=None, scale=KEY_DIM ** -0.5, *,
                   max_nodes=abi.DRAFT_MAX_NODES, output_dtype=None, steps=None):
    """One tree-attention call (arguments as `TreeAttention.bind`); returns [rows, heads, 512]."""
    import torch

    op = TreeAttention(torch, batch=int(seq_lens.shape[0]), heads=int(query.shape[1]), max_nodes=max_nodes,
                       max_tokens=int(query.shape[0]), max_context=int(block_table.shape[1]) * BLOCK_TOKENS,
                       device=query.device, output_dtype=output_dtype)
    return op.bind(query, kv_cache, block_table, seq_lens, cu_seqlens, visible, scale, steps=steps)()
