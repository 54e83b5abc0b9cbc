"""Verification of drafted tokens: `kvip_amd.DraftVerifier`.

Chains drawn from a draft distribution (`draft_probs`) and chains or trees of chosen tokens are walked
against the target's probabilities by given random numbers, so that the tokens that come out are
distributed as the target alone would draw them; `include/kvip_hip_draft.h` states the rules. The path and
the number of rows kept go to `kvip_amd.PageTables.commit`. Nothing is read back or allocated by a call, so a
round can be captured; the random numbers are inputs. The reference has no counterpart.
"""
from __future__ import annotations

from kvip_amd.runtime import abi


class DraftVerifier:
    """out_tokens int64 [batch, max_nodes], kept int32 [batch], path int32 [batch, max_nodes] and status are allocated
    once; `bind` validates a call's tensors, `__call__` enqueues it on the current stream (one object's calls
    follow one another, as they share its workspace)."""

    def __init__(self, torch, *, batch, max_nodes, vocab, device):
        abi.require(1 <= batch <= abi.DRAFT_MAX_BATCH, f"batch must be in 1..{abi.DRAFT_MAX_BATCH}")
        abi.require(1 <= max_nodes <= abi.DRAFT_MAX_NODES, f"max_nodes must be in 1..{abi.DRAFT_MAX_NODES}")
        abi.require(1 <= vocab <= 1 << 20, "vocab must be in 1..2^20")
        self.torch, self.device = torch, abi.device_of(torch, device)
        abi.require(self.device.type == "cuda", "verification runs on the GPU (kvip_amd has no CPU path)")
        self.batch, self.max_nodes, self.vocab = int(batch), int(max_nodes), int(vocab)
        self.library = abi.load_library()
        self.out_tokens = torch.full((batch, max_nodes), -1, dtype=torch.int64, device=self.device)
        self.kept = torch.zeros(batch, dtype=torch.int32, device=self.device)
        self.path = torch.full((batch, max_nodes), -1, dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        nbytes = int(self.library.kvip_hip_verify_drafts_workspace_bytes(batch, vocab))
        self.workspace = torch.zeros(nbytes // 8, dtype=torch.int64, device=self.device)
        self.args = None

    def bind(self, probs, tokens, cu_seqlens, uniforms, final_uniforms, *, parents=None, draft_probs=None, steps=None):
        """probs [rows, vocab] (fp32, bf16 or fp16; rows at any stride): the target's probabilities after
        each step token; tokens int64 [rows]; cu_seqlens int32 [batch + 1]; uniforms float32 [rows] and
        final_uniforms float32 [batch] in [0, 1). parents int32 [rows]: trees of chosen tokens; draft_probs (as
        probs): a chain whose next token each row drew; neither: a chain of chosen tokens. steps int32 [batch]
        (PageTables.steps, read before its commit): requests with 0, which extend refused, keep nothing."""
        t = self.torch
        codes = {t.float32: abi.DTYPE_FP32, t.bfloat16: abi.DTYPE_BF16, t.float16: abi.DTYPE_FP16}
        rows = int(probs.shape[0])
        abi.require(probs.dtype in codes, "probs must be float32, bfloat16 or float16")
        abi.require(1 <= rows <= abi.DRAFT_MAX_TOKENS, f"probs must have 1..{abi.DRAFT_MAX_TOKENS} rows")
        abi.require(parents is None or draft_probs is None, "draft_probs go with a chain, not with parents")
        for x, what in ((probs, "probs"), (draft_probs, "draft_probs")):
            abi.require(x is None or (x.dtype == probs.dtype and tuple(x.shape) == (rows, self.vocab) and
                                      (self.vocab == 1 or x.stride(1) == 1) and (rows == 1 or x.stride(0) >= self.vocab) and
                                      x.device == self.device),
                        f"{what} must be {probs.dtype} [{rows}, {self.vocab}] with contiguous rows on {self.device}")
        for x, dtype, shape, what in ((tokens, t.int64, (rows,), "tokens"), (uniforms, t.float32, (rows,), "uniforms"),
                                      (cu_seqlens, t.int32, (self.batch + 1,), "cu_seqlens"),
                                      (final_uniforms, t.float32, (self.batch,), "final_uniforms"),
                                      (parents, t.int32, (rows,), "parents"), (steps, t.int32, (self.batch,), "steps")):
            abi.require(x is None and what in ("parents", "steps") or
                        (x.dtype == dtype and tuple(x.shape) == shape and x.is_contiguous() and x.device == self.device),
                        f"{what} must be contiguous {dtype} {list(shape)} on {self.device}")
        p = abi.ptr
        self.args = abi.VerifyArgs(
            probs=p(probs), draft_probs=p(draft_probs), tokens=p(tokens), cu_seqlens=p(cu_seqlens), parents=p(parents),
            uniforms=p(uniforms), final_uniforms=p(final_uniforms), out_tokens=p(self.out_tokens), kept=p(self.kept),
            path=p(self.path), workspace=p(self.workspace), status=p(self.status),
            probs_stride=max(probs.stride(0), self.vocab), draft_stride=0 if draft_probs is None else
            max(draft_probs.stride(0), self.vocab), batch=self.batch, max_nodes=self.max_nodes, max_tokens=rows,
            vocab=self.vocab, dtype=codes[probs.dtype], steps=p(steps))
        self._bound = (probs, draft_probs, tokens, cu_seqlens, parents, uniforms, final_uniforms, steps)
        return self

    def __call__(self):
        """Returns (out_tokens, kept, path)."""
        abi.require(self.args is not None, "bind() the step's tensors first")
        abi.launch(self.torch, self.device, self.library.kvip_hip_verify_drafts, self.args, "verification")
        return self.out_tokens, self.kept, self.path
