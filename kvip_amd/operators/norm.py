"""Queries and keys normed per head and turned by their positions in one pass: `kvip_amd.NormRotary`.

What stands between a projection and attention where heads are normed: a norm over each head's features
(root mean square, or mean and variance), its weight and bias, and the turn of `kvip_amd.Rotary`, in one reading. For the
lightning indexer (`kvip_amd.PrefillIndexer`, `kvip_amd.LIFetch`) the heads leave as fp8 with a scale each, keys
into their paged cache. `bind` validates a call's tensors, the call only enqueues (capturable).
`include/kvip_hip_prompt.h` states the arithmetic. The reference leaves these steps to its engine.
"""
from __future__ import annotations

import math

from kvip_amd.operators.rotary import _dtype_code
from kvip_amd.runtime import abi

BLOCK_TOKENS = 128
INDEX_DIM = 128
_NORMS = {None: abi.NORM_NONE, "rms": abi.NORM_RMS, "layer": abi.NORM_LAYER}


def _rows_apart(tokens, heads, dim, by_token, by_head):
    """Whether the rows [tokens, heads] of dim elements at these strides lie apart."""
    return (heads <= 1 or by_head >= dim) and (tokens <= 1 or by_token >= dim) and (
        tokens <= 1 or heads <= 1 or by_token >= by_head * (heads - 1) + dim or by_head >= by_token * (tokens - 1) + dim)


class NormRotary:
    """rotary: the `kvip_amd.Rotary` whose layout, angles and device are taken; dim: features of a head (at least its
    rotary_dim, at most 512); query_norm and key_norm: None, "rms" or "layer". status collects device-side problems."""

    def __init__(self, torch, *, rotary, dim, query_norm=None, key_norm=None, epsilon=1e-6):
        abi.require(query_norm in _NORMS and key_norm in _NORMS, 'a norm is None, "rms" or "layer"')
        abi.require(rotary.rotary_dim <= dim <= abi.NORM_MAX_DIM, f"dim must be in rotary_dim..{abi.NORM_MAX_DIM}")
        abi.require(math.isfinite(epsilon) and epsilon >= 0, "epsilon must be finite and not negative")
        self.torch, self.rotary, self.device = torch, rotary, rotary.device
        self.dim, self.epsilon, self.norms = int(dim), float(epsilon), (_NORMS[query_norm], _NORMS[key_norm])
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.library = abi.load_library()
        self.args = None

    def _heads(self, x, tokens, what):
        """[tokens, heads, dim] of an array with one head or more, checked."""
        abi.require(x.dim() in (2, 3) and x.shape[0] == tokens and x.shape[-1] == self.dim,
                    f"{what} must be [{tokens}, heads, {self.dim}] or [{tokens}, {self.dim}]")
        x = x if x.dim() == 3 else x[:, None]
        abi.require(x.stride(2) == 1 or self.dim == 1, f"{what}: the last dimension must be contiguous")
        abi.require(x.device == self.device, f"{what} must be on {self.device}")
        abi.require(1 <= x.shape[1] <= 65536, f"{what} must have 1..65536 heads")
        return x

    def _tensor(self, x, weight, bias, norm, tokens, what):
        for w, name in ((weight, "weight"), (bias, "bias")):
            abi.require(w is None or (w.dtype == self.torch.float32 and tuple(w.shape) == (self.dim,) and w.is_contiguous() and
                                      w.device == self.device),
                        f"{what}_{name} must be contiguous float32 [{self.dim}] on {self.device}")
        x = self._heads(x, tokens, what)
        return x, abi.NormTensor(x=abi.ptr(x), weight=abi.ptr(weight), bias=abi.ptr(bias), x_token=x.stride(0),
                                 x_head=x.stride(1), heads=int(x.shape[1]), norm=norm)

    def _apart(self, y, tokens, what):
        abi.require(_rows_apart(tokens, int(y.shape[1]), self.dim, y.stride(0), y.stride(1)), f"{what}: output rows must not overlap")

    def _output(self, tensor, x, out, tokens, what):
        y = self._heads(out, tokens, what + "_out")
        abi.require(y.shape == x.shape and y.dtype == x.dtype, f"{what} and its output must have one shape and type")
        abi.require(y.data_ptr() != x.data_ptr() or y.stride() == x.stride(), f"{what}: an array normed in place keeps its strides")
        self._apart(y, tokens, what)
        tensor.out, tensor.out_token, tensor.out_head = abi.ptr(y), y.stride(0), y.stride(1)

    def _codes(self, tensor, x, out, scale, tokens):
        t = self.torch
        abi.require(out is not None and scale is not None, "quantised queries need query_out and query_scale")
        y = self._heads(out, tokens, "query_out")
        abi.require(y.shape == x.shape and y.dtype in (t.float8_e4m3fn, t.uint8), "query_out must be float8_e4m3fn, of the query's shape")
        abi.require(scale.dtype == t.float32 and tuple(scale.shape) == tuple(x.shape[:2]) and scale.is_contiguous() and
                    scale.device == self.device, f"query_scale must be contiguous float32 {list(x.shape[:2])} on {self.device}")
        abi.require(all(v % 4 == 0 for v in (y.data_ptr(), y.stride(0), y.stride(1))),
                    "query_out: address and strides must be multiples of 4 bytes")
        self._apart(y, tokens, "query")
        tensor.out, tensor.out_token, tensor.out_head, tensor.scales = abi.ptr(y), y.stride(0), y.stride(1), abi.ptr(scale)

    def _pages(self, tensor, x, slots, cache, scales, tokens):
        t = self.torch
        abi.require(slots is not None and cache is not None and scales is not None,
                    "quantised keys need slots, key_cache and key_scales")
        abi.require(x.shape[1] == 1, "quantised keys have one head")
        abi.require(slots.dtype == t.int64 and tuple(slots.shape) == (tokens,) and slots.is_contiguous() and
                    slots.device == self.device, f"slots must be contiguous int64 [{tokens}] on {self.device}")
        abi.require(cache.dtype in (t.float8_e4m3fn, t.uint8) and cache.dim() == 3 and cache.shape[0] >= 1 and
                    tuple(cache.shape[1:]) == (BLOCK_TOKENS, INDEX_DIM) and tuple(cache.stride()[1:]) == (INDEX_DIM, 1) and
                    (cache.shape[0] == 1 or cache.stride(0) >= BLOCK_TOKENS * INDEX_DIM) and cache.device == self.device,
                    f"key_cache must be float8_e4m3fn [blocks, 128, 128] of contiguous blocks on {self.device}")
        abi.require(scales.dtype == t.float32 and tuple(scales.shape) == (cache.shape[0], BLOCK_TOKENS) and
                    scales.stride(1) == 1 and (cache.shape[0] == 1 or scales.stride(0) >= BLOCK_TOKENS) and
                    scales.device == self.device, f"key_scales must be float32 [blocks, 128] on {self.device}")
        abi.require(cache.data_ptr() % 4 == 0 and cache.stride(0) % 4 == 0, "key_cache: address and strides must be multiples of 4 bytes")
        tensor.out, tensor.out_token = abi.ptr(cache), max(cache.stride(0), BLOCK_TOKENS * INDEX_DIM)
        tensor.scales, tensor.out_head = abi.ptr(scales), max(scales.stride(0), BLOCK_TOKENS)

    def bind(self, positions, query, key=None, *, query_weight=None, query_bias=None, key_weight=None, key_bias=None,
             query_out=None, key_out=None, query_scale=None, slots=None, key_cache=None, key_scales=None):
        """positions int64 [tokens]; query (and key) [tokens, heads, dim] or [tokens, dim] of one type (bf16, fp16, fp32),
        strided as long as the last dimension is contiguous; weights and biases float32 [dim]. Without an output the
        array is normed in place. An output does not overlap another array.
        For the indexer (heads of 128): query_out float8_e4m3fn like the query with query_scale float32 [tokens, heads],
        and the key, of one head, goes to slots int64 [tokens] (page * 128 + row, negative: none; no slot twice) of
        key_cache float8_e4m3fn [blocks, 128, 128] and key_scales float32 [blocks, 128]."""
        t = self.torch
        abi.require(positions.dtype == t.int64 and positions.dim() == 1 and positions.is_contiguous() and
                    positions.device == self.device, f"positions must be contiguous int64 [tokens] on {self.device}")
        tokens = int(positions.shape[0])
        abi.require(key is None or key.dtype == query.dtype, "key must have the query's type")
        abi.require(key is not None or (key_weight is None and key_bias is None and key_out is None and slots is None and
                                        key_cache is None and key_scales is None), "what is the key's needs a key")
        quantised = query_scale is not None or slots is not None or key_cache is not None or key_scales is not None
        rotary = self.rotary
        args = abi.NormRotaryArgs(positions=abi.ptr(positions), frequencies=abi.ptr(rotary.frequencies), slots=abi.ptr(slots),
                                  status=abi.ptr(self.status), tokens=tokens, dim=self.dim, rotary_dim=rotary.rotary_dim,
                                  half=int(rotary.half), dtype=_dtype_code(t, query.dtype, "query"), quantised=int(quantised),
                                  num_blocks=0 if key_cache is None else int(key_cache.shape[0]), epsilon=self.epsilon,
                                  magnitude=rotary.magnitude)
        x, tensor = self._tensor(query, query_weight, query_bias, self.norms[0], tokens, "query")
        if quantised:
            abi.require(self.dim == INDEX_DIM, f"quantised heads have {INDEX_DIM} features")
            abi.require(key_out is None, "quantised keys go to key_cache, not to key_out")
            self._codes(tensor, x, query_out, query_scale, tokens)
        else:
            query_out = query if query_out is None else query_out
            self._output(tensor, x, query_out, tokens, "query")
        args.tensors[0] = tensor
        if key is not None:
            x, tensor = self._tensor(key, key_weight, key_bias, self.norms[1], tokens, "key")
            if quantised:
                self._pages(tensor, x, slots, key_cache, key_scales, tokens)
                key_out = key_cache
            else:
                key_out = key if key_out is None else key_out
                self._output(tensor, x, key_out, tokens, "key")
            args.tensors[1] = tensor
        self.args, self._outputs = args, (query_out, key_out)
        self._bound = (positions, query, key, query_weight, query_bias, key_weight, key_bias, query_out, key_out, query_scale,
                       slots, key_cache, key_scales, rotary)
        return self

    def __call__(self):
        """Returns (query output, key output, key cache or None)."""
        abi.require(self.args is not None, "bind() the heads first")
        if self.args.tokens:
            abi.launch(self.torch, self.device, self.library.kvip_hip_norm_rotary, self.args, "norm and rotation")
        return self._outputs
