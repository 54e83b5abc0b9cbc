"""Page tables of a batch on the GPU: `kvip_amd.PageTables`.

Holds, as device tensors, the block table and length of every request and the stack of free pages
of a paged cache, and lays out a step from the request lengths without a host read: `extend(counts)`
appends tokens (pages, slots, positions, the visibility of a tree's tokens), `commit(kept)` keeps the
accepted ones and gives the other pages back, `truncate(lengths)` shortens or ends requests. The
tensors feed the operators of the same step: `cu_seqlens`, `lengths`, `block_table`, `visible` and `steps` go to
`kvip_amd.TreeAttention`, `slots` and `positions` to `kvip_amd.KvRowStore` and `kvip_amd.Rotary`. Steps of chains (and
prompt chunks) also feed the selection: `block_table`, `lengths` and `cu_seqlens` go to `kvip_amd.PrefillIndexer`, `slots` to
`kvip_amd.IndexCacheStorage` as its slot mapping. Trees do not: that indexer lets a row see every row of the step before
it, siblings among them, and siblings share a position. `include/kvip_hip_draft.h` states the rules. Calls only
enqueue on the current stream and allocate nothing, so they can be captured; one object's calls follow one
another (they share its state). There is no CPU path and no counterpart in the reference, whose engine does this on the host.
"""
from __future__ import annotations

import ctypes

from kvip_amd.runtime import abi

BLOCK_TOKENS = 128


class PageTables:
    """batch: requests (1..1024, a request that is not there has length 0); max_context: positions of a
    request; num_blocks: pages of the cache, all free at first and taken from 0 up; max_tokens: rows
    of a step; caches: the paged tensors [num_blocks, 128, ...] (rows contiguous, a multiple of 4
    bytes, none over another) whose rows `commit(kept, path)` copies together: the KV rows, index keys and
    scales of every layer.

    block_table int32 [batch, blocks], lengths int32 [batch], free int32 [num_blocks] and free_count int32
    [1] are the state; steps int32 [batch] has the tokens that the last extend appended (0 where it refused a
    request, whose rows stay in the step: TreeAttention and DraftVerifier take `steps` to leave it out); cu_seqlens
    int32 [batch + 1], positions, slots, visible int64 [max_tokens] the last step's layout; status int32 [1] collects
    KVIP_STATUS_* bits."""

    def __init__(self, torch, *, batch, max_context, num_blocks, max_tokens, device, caches=()):
        abi.require(1 <= batch <= abi.DRAFT_MAX_BATCH, f"batch must be in 1..{abi.DRAFT_MAX_BATCH}")
        abi.require(1 <= max_context <= 1 << 24, "max_context must be in 1..2^24")
        abi.require(1 <= num_blocks < 1 << 24, "num_blocks must be in 1..2^24 - 1")
        abi.require(1 <= max_tokens <= abi.DRAFT_MAX_TOKENS, f"max_tokens must be in 1..{abi.DRAFT_MAX_TOKENS}")
        self.torch, self.device = torch, abi.device_of(torch, device)
        abi.require(self.device.type == "cuda", "page tables live on the GPU (kvip_amd has no CPU path)")
        self.batch, self.num_blocks, self.max_tokens = int(batch), int(num_blocks), int(max_tokens)
        self.max_blocks = (int(max_context) + BLOCK_TOKENS - 1) // BLOCK_TOKENS
        rows = [self._rows(c) for c in caches]
        abi.require(len({base for base, *_ in rows}) == len(rows), "a cache must not be named twice")
        self.caches = tuple(caches)

        def ints(*shape, dtype=torch.int32):
            return torch.zeros(shape, dtype=dtype, device=self.device)

        self.block_table = ints(self.batch, self.max_blocks).fill_(-1)
        self.lengths = ints(self.batch)
        self.free = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=self.device)
        self.free_count = ints(1).fill_(num_blocks)
        self.bases, self.steps, self.ticket, self.status = ints(self.batch), ints(self.batch), ints(1), ints(1)
        self.cu_seqlens = ints(self.batch + 1)
        self.positions, self.slots, self.visible = (ints(self.max_tokens, dtype=torch.int64) for _ in range(3))
        self.slots.fill_(-1)
        self.rows = torch.tensor(rows, dtype=torch.int64, device=self.device) if rows else None
        self.library = abi.load_library()
        p = abi.ptr
        self._args = abi.PageTableArgs(
            block_table=p(self.block_table), lengths=p(self.lengths), free_pages=p(self.free), free_count=p(self.free_count),
            bases=p(self.bases), steps=p(self.steps), ticket=p(self.ticket), rows=p(self.rows), cu_seqlens=p(self.cu_seqlens),
            positions=p(self.positions), slots=p(self.slots), visible=p(self.visible), status=p(self.status),
            batch=self.batch, max_blocks=self.max_blocks, num_blocks=self.num_blocks, max_tokens=self.max_tokens,
            row_sets=len(rows))

    def _rows(self, cache):
        """(base, block stride, row stride, row bytes) of a paged tensor, in bytes."""
        size = cache.element_size()
        abi.require(cache.device == self.device, "a cache must be on the tables' device")
        abi.require(cache.dim() >= 2 and cache.shape[0] >= self.num_blocks and cache.shape[1] == BLOCK_TOKENS,
                    f"a cache must be [{self.num_blocks} or more, {BLOCK_TOKENS}, ...]")
        width = 1
        for n, stride in zip(reversed(cache.shape[2:]), reversed(cache.stride()[2:])):
            abi.require(n == 1 or stride == width, "a cache's rows must be contiguous")
            width *= n
        found = (cache.data_ptr(), cache.stride(0) * size, cache.stride(1) * size, width * size)
        abi.require(all(v % 4 == 0 for v in found) and width >= 1,
                    "a cache's address, strides and rows must be multiples of 4 bytes")
        _, block, row, size = found
        places, pages = row * (BLOCK_TOKENS - 1), block * (self.num_blocks - 1)  # from the first to the last
        apart = row >= size and (self.num_blocks == 1 or block >= places + size or (block >= size and row >= pages + size))
        abi.require(apart, "a cache's rows must not overlap")
        return found

    def _ints(self, x, shape, what):
        abi.require(x.dtype == self.torch.int32 and tuple(x.shape) == shape and x.is_contiguous() and x.device == self.device,
                    f"{what} must be contiguous int32 {list(shape)} on {self.device}")
        return x.data_ptr()

    def extend(self, counts, parents=None):
        """Appends counts[b] tokens to request b; counts int32 [batch] on the device. parents int32
        [max_tokens] names every row's parent within its request (-1: none) where the tokens are trees of
        at most 64: positions then follow the depth. `visible` gets each token's ancestors and itself: in a chain
        (no parents) the tokens before it and itself.
        Returns (cu_seqlens, slots, positions)."""
        a = self._args  # copied by the launch
        a.counts = self._ints(counts, (self.batch,), "counts")
        a.parents = 0 if parents is None else self._ints(parents, (self.max_tokens,), "parents")
        abi.launch(self.torch, self.device, self.library.kvip_hip_page_tables_extend, a, "page tables")
        return self.cu_seqlens, self.slots, self.positions

    def commit(self, kept, path=None):
        """Keeps kept[b] tokens of the last step (int32 [batch], at most those appended) and gives back
        the pages of the rest. path int32 [batch, places], as kvip_amd.DraftVerifier returns it, names the
        kept tokens of trees: their rows in `caches` are copied together first (without it the first
        kept[b] are kept; more kept than places set a status bit). Returns lengths."""
        a = self._args  # copied by the launch
        a.targets, a.kept = self._ints(kept, (self.batch,), "kept"), 1
        if path is not None:
            abi.require(path.dim() == 2 and path.shape[1] >= 1, f"path must be int32 [{self.batch}, places]")
            a.path, a.path_stride = self._ints(path, (self.batch, int(path.shape[1])), "path"), int(path.shape[1])
            abi.launch(self.torch, self.device, self.library.kvip_hip_page_tables_move, a, "kept rows")
        abi.launch(self.torch, self.device, self.library.kvip_hip_page_tables_truncate, a, "page tables")
        return self.lengths

    def truncate(self, lengths):
        """Cuts request b to lengths[b] tokens (int32 [batch] on the device; one that is not shorter
        sets a status bit where it is longer) and gives back the pages that nothing needs; 0 ends a
        request. Pages come back in the order that undoes an `extend` from these lengths. Returns lengths."""
        a = self._args  # copied by the launch
        a.targets, a.kept = self._ints(lengths, (self.batch,), "lengths"), 0
        abi.launch(self.torch, self.device, self.library.kvip_hip_page_tables_truncate, a, "page tables")
        return self.lengths
