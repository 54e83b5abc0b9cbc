"""From logits to the probabilities that tokens are drawn from or drafts verified against:
`kvip_amd.LogitProcessor`, and the histories that its penalties read: `kvip_amd.TokenHistory`.

Penalties for tokens that a request holds already (its prompt's, those it wrote, and the drafted ones on the way to a
row), biases per request, grammar masks per row, temperature and softmax, in two passes over the logits. The
probabilities go to `kvip_amd.DraftVerifier`; the tokens that come out of it, to `TokenHistory.append`. Both bind
or check their tensors and only enqueue (capturable). `include/kvip_hip_prompt.h` states the rules. The reference
leaves these steps to its engine.
"""
from __future__ import annotations

from kvip_amd.runtime import abi


def _codes(torch):
    return {torch.float32: abi.DTYPE_FP32, torch.bfloat16: abi.DTYPE_BF16, torch.float16: abi.DTYPE_FP16}


class TokenHistory:
    """counts int32 [batch, vocab] (how often a request wrote a token), seen int32 [batch, (vocab + 31) / 32] (bits: it
    wrote the token or its prompt has it) and status, allocated once and empty. Calls may come from several threads and
    streams as long as they are for different requests."""

    def __init__(self, torch, *, batch, vocab, device):
        abi.require(1 <= batch <= abi.DRAFT_MAX_BATCH, f"batch must be in 1..{abi.DRAFT_MAX_BATCH}")
        abi.require(1 <= vocab <= 1 << 20, "vocab must be in 1..2^20")
        self.torch, self.device = torch, abi.device_of(torch, device)
        abi.require(self.device.type == "cuda", "histories are kept on the GPU (kvip_amd has no CPU path)")
        self.batch, self.vocab = int(batch), int(vocab)
        self.library = abi.load_library()
        self.counts = torch.zeros((batch, vocab), dtype=torch.int32, device=self.device)
        self.seen = torch.zeros((batch, (vocab + 31) // 32), dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        p = abi.ptr
        self._args = abi.HistoryArgs(counts=p(self.counts), seen=p(self.seen), status=p(self.status), batch=self.batch,
                                     vocab=self.vocab)

    def _check(self, x, dtype, shape, what):
        # Worded only where it fails: with a message made for every check a call took 9.4 us of the host instead of 6.4.
        if x.dtype is not dtype or x.shape != shape or not x.is_contiguous() or x.device != self.device:
            raise ValueError(f"{what} must be contiguous {dtype} {list(shape)} on {self.device}")
        return x.data_ptr()

    def load(self, requests, tokens, cu_seqlens, prompt_lens):
        """Replaces what requests[i] (int32 [n] in 0 .. batch - 1, none twice; negative: none) holds by the tokens
        cu_seqlens[i] .. cu_seqlens[i + 1] (int64, packed), the first prompt_lens[i] (int32 [n]) of which are its
        prompt; no tokens: it holds none. Returns counts."""
        t = self.torch
        n = requests.numel()
        if requests.dim() != 1 or not 1 <= n <= abi.DRAFT_MAX_BATCH:
            raise ValueError(f"requests must be int32 [1..{abi.DRAFT_MAX_BATCH}]")
        abi.require(tokens.dim() == 1 and tokens.numel() <= 0x7FFFFFFF, "tokens must be int64 [up to 2^31 - 1]")
        a = abi.HistoryArgs.from_buffer_copy(self._args)  # this call's: the entry runs without the interpreter's lock
        a.requests, a.count = self._check(requests, t.int32, (n,), "requests"), n
        a.cu_seqlens = self._check(cu_seqlens, t.int32, (n + 1,), "cu_seqlens")
        a.prompt_lens = self._check(prompt_lens, t.int32, (n,), "prompt_lens")
        a.max_tokens = tokens.numel()
        # Without tokens nothing is read: any address that is not null.
        a.tokens = self._check(tokens, t.int64, (a.max_tokens,), "tokens") or a.counts
        abi.launch(t, self.device, self.library.kvip_hip_history_load, a, "token history")
        return self.counts

    def append(self, tokens, kept):
        """Adds the first kept[b] (int32 [batch]) of tokens[b] (int64 [batch, up to 64]) to request b, as
        `kvip_amd.DraftVerifier` returns them. Returns counts."""
        t = self.torch
        places = tokens.shape[1] if tokens.dim() == 2 else 0
        if not 1 <= places <= abi.DRAFT_MAX_NODES:
            raise ValueError(f"tokens must be int64 [{self.batch}, 1..{abi.DRAFT_MAX_NODES}]")
        a = abi.HistoryArgs.from_buffer_copy(self._args)  # this call's: the entry runs without the interpreter's lock
        a.tokens, a.token_stride = self._check(tokens, t.int64, (self.batch, places), "tokens"), places
        a.kept = self._check(kept, t.int32, (self.batch,), "kept")
        abi.launch(t, self.device, self.library.kvip_hip_history_append, a, "token history")
        return self.counts


class LogitProcessor:
    """probs [max_tokens, vocab] (float32 unless output_dtype says bf16 or fp16), status and workspace allocated once;
    `bind` validates a call's tensors, `__call__` enqueues it on the current stream (one object's calls follow one
    another, as they share its workspace)."""

    def __init__(self, torch, *, batch, max_tokens, vocab, device, output_dtype=None):
        abi.require(1 <= batch <= abi.DRAFT_MAX_BATCH, f"batch must be in 1..{abi.DRAFT_MAX_BATCH}")
        abi.require(1 <= max_tokens <= abi.DRAFT_MAX_TOKENS, f"max_tokens must be in 1..{abi.DRAFT_MAX_TOKENS}")
        abi.require(1 <= vocab <= 1 << 20, "vocab must be in 1..2^20")
        output_dtype = torch.float32 if output_dtype is None else output_dtype
        abi.require(output_dtype in _codes(torch), "probabilities are float32, bfloat16 or float16")
        self.torch, self.device = torch, abi.device_of(torch, device)
        abi.require(self.device.type == "cuda", "logits are processed on the GPU (kvip_amd has no CPU path)")
        self.batch, self.max_tokens, self.vocab = int(batch), int(max_tokens), int(vocab)
        self.library = abi.load_library()
        nbytes = int(self.library.kvip_hip_process_logits_workspace_bytes(max_tokens, vocab))
        abi.require(nbytes > 0, "max_tokens * vocab is too large for one call")
        self.probs = torch.zeros((max_tokens, vocab), dtype=output_dtype, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self.args = None

    def bind(self, logits, cu_seqlens, *, temperature=None, history=None, repetition=None, presence=None, frequency=None,
             tokens=None, visible=None, bias_tokens=None, bias_values=None, allowed=None):
        """logits [max_tokens, vocab] (fp32, bf16 or fp16; rows at any stride); cu_seqlens int32 [batch + 1]: request b's
        rows. float32 [batch] each: temperature (not above 0: the largest logit's token), repetition, presence and
        frequency penalties, which read `history` (a TokenHistory of this batch and vocabulary) and, for drafted rows,
        tokens int64 [max_tokens] with visible int64 [max_tokens] as kvip_amd.PageTables.extend writes it: the
        drafted tokens on the way to a row count as written, a request's token 0 being in its history. bias_tokens int32
        and bias_values float32 [batch, n] (n up to 4096; a token that is negative: none; one that is named
        twice gets both). allowed int32 [max_tokens, (vocab + 31) / 32]: bit v % 32 of word v / 32 allows token v."""
        t, codes = self.torch, _codes(self.torch)
        abi.require(logits.dtype in codes and tuple(logits.shape) == (self.max_tokens, self.vocab) and
                    (self.vocab == 1 or logits.stride(1) == 1) and (self.max_tokens == 1 or logits.stride(0) >= self.vocab) and
                    logits.device == self.device,
                    f"logits must be float32, bfloat16 or float16 [{self.max_tokens}, {self.vocab}] with contiguous rows on {self.device}")
        begin, end = logits.data_ptr(), logits.data_ptr() + ((self.max_tokens - 1) * logits.stride(0) + self.vocab) * logits.element_size()
        own, own_end = self.probs.data_ptr(), self.probs.data_ptr() + self.probs.numel() * self.probs.element_size()
        abi.require(end <= own or own_end <= begin, "logits must not be this object's probabilities")
        abi.require(history is None or (history.batch == self.batch and history.vocab == self.vocab and
                                        history.device == self.device), "history must be of this batch, vocabulary and device")
        abi.require((tokens is None) == (visible is None), "tokens go with visible")
        abi.require((bias_tokens is None) == (bias_values is None), "bias_tokens go with bias_values")
        biases = 0 if bias_tokens is None else int(bias_tokens.shape[1]) if bias_tokens.dim() == 2 else -1
        abi.require(0 <= biases <= abi.LOGIT_MAX_BIASES, f"bias_tokens must be int32 [{self.batch}, up to {abi.LOGIT_MAX_BIASES}]")
        words = (self.vocab + 31) // 32
        for x, dtype, shape, what in (
                (cu_seqlens, t.int32, (self.batch + 1,), "cu_seqlens"), (temperature, t.float32, (self.batch,), "temperature"),
                (repetition, t.float32, (self.batch,), "repetition"), (presence, t.float32, (self.batch,), "presence"),
                (frequency, t.float32, (self.batch,), "frequency"), (tokens, t.int64, (self.max_tokens,), "tokens"),
                (visible, t.int64, (self.max_tokens,), "visible"), (bias_tokens, t.int32, (self.batch, biases), "bias_tokens"),
                (bias_values, t.float32, (self.batch, biases), "bias_values"),
                (allowed, t.int32, (self.max_tokens, words), "allowed")):
            abi.require(x is None and what != "cu_seqlens" or
                        (x.dtype == dtype and tuple(x.shape) == shape and x.is_contiguous() and x.device == self.device),
                        f"{what} must be contiguous {dtype} {list(shape)} on {self.device}")
        p = abi.ptr
        self.args = abi.LogitArgs(
            logits=p(logits), probs=p(self.probs), cu_seqlens=p(cu_seqlens), temperature=p(temperature), repetition=p(repetition),
            presence=p(presence), frequency=p(frequency), counts=0 if history is None else p(history.counts),
            seen=0 if history is None else p(history.seen), tokens=p(tokens), visible=p(visible),
            bias_tokens=p(bias_tokens) if biases else 0, bias_values=p(bias_values) if biases else 0, allowed=p(allowed),
            workspace=p(self.workspace), status=p(self.status), logits_stride=max(logits.stride(0), self.vocab),
            probs_stride=self.vocab, batch=self.batch, max_tokens=self.max_tokens, vocab=self.vocab, biases=biases,
            dtype=codes[logits.dtype], probs_dtype=codes[self.probs.dtype])
        self._bound = (logits, cu_seqlens, temperature, history, repetition, presence, frequency, tokens, visible, bias_tokens,
                       bias_values, allowed)
        return self

    def __call__(self):
        """Returns probs."""
        abi.require(self.args is not None, "bind() the step's tensors first")
        abi.launch(self.torch, self.device, self.library.kvip_hip_process_logits, self.args, "logits")
        return self.probs
