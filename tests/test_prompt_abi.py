"""The C ABI and the Python checks of the operators around a prompt chunk's layers, without a GPU: exported symbols,
struct layouts, arguments rejected before any launch."""
import ctypes
import re
import subprocess
import textwrap

import pytest

import kvip_amd
from kvip_amd.runtime import abi
from tests.conftest import ROOT
from tests.test_draft_abi import rejects

HEADER = ROOT / "include" / "kvip_hip_prompt.h"
STRUCTS = {
    "KvipChunkAttnArgs": abi.ChunkAttnArgs,
    "KvipNormTensor": abi.NormTensor,
    "KvipNormRotaryArgs": abi.NormRotaryArgs,
    "KvipHistoryArgs": abi.HistoryArgs,
    "KvipLogitArgs": abi.LogitArgs,
}


def test_every_declared_symbol_is_exported():
    lib = abi.load_library()
    names = set(re.findall(r"^\s*uint(?:32|64)_t\s+(kvip_hip_\w+)\s*\(", HEADER.read_text(), re.M))
    assert names == set(abi.PROMPT_PROTOTYPES)
    assert all(hasattr(lib, name) for name in names)
    assert lib.kvip_hip_prompt_abi_version() == abi.PROMPT_ABI_VERSION
    defines = dict(re.findall(r"#define KVIP_(\w+) (\d+)u?\b", HEADER.read_text()))
    for name in ("PROMPT_ABI_VERSION", "NORM_NONE", "NORM_RMS", "NORM_LAYER", "NORM_MAX_DIM", "LOGIT_MAX_BIASES"):
        assert int(defines[name]) == getattr(abi, name), name


def test_ctypes_layout_matches_c(tmp_path):
    assert set(re.findall(r"typedef struct (\w+)", HEADER.read_text())) == set(STRUCTS)
    lines = []
    for cname, cls in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {field} %zu\\n", offsetof({cname}, {field}));' for field, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text(textwrap.dedent('#include <stddef.h>\n#include <stdio.h>\n#include "kvip_hip_prompt.h"\nint main(void){\n'
                                   + "\n".join(lines) + "\nreturn 0;}\n"))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    layout = {(a, b): int(c) for a, b, c in (line.split() for line in out if line)}
    for cname, cls in STRUCTS.items():
        assert layout[(cname, "size")] == ctypes.sizeof(cls), cname
        for field, _ in cls._fields_:
            assert layout[(cname, field)] == getattr(cls, field).offset, (cname, field)


def test_chunk_attention_rejects_before_launch():
    good = dict({f: 256 for f, _ in abi.ChunkAttnArgs._fields_[:10]}, kv_block_stride=128 * 656, row_stride=656, batch=2,
                heads=16, max_tokens=8, max_rows=512, max_blocks=4, num_blocks=8, output_dtype=abi.DTYPE_BF16, scale=1.0)
    rejects("kvip_hip_chunk_attention", abi.ChunkAttnArgs, good, [
        dict(query=0), dict(query=264), dict(kv_cache=264), dict(output=260), dict(workspace=0), dict(workspace=264),
        dict(seq_lens=0), dict(cu_seqlens=0), dict(block_table=0), dict(batch=0), dict(batch=1025), dict(heads=0),
        dict(heads=129), dict(max_tokens=0), dict(max_tokens=(1 << 20) + 1), dict(max_rows=0), dict(max_rows=(1 << 31) + 1),
        dict(max_blocks=0), dict(max_blocks=(1 << 17) + 1), dict(num_blocks=0), dict(num_blocks=1 << 24), dict(row_stride=640),
        dict(row_stride=664), dict(kv_block_stride=128 * 640), dict(kv_block_stride=128 * 656 + 8),
        dict(output_dtype=abi.DTYPE_FP16), dict(row_stride=(1 << 24) + 16, kv_block_stride=1 << 32),
        dict(scale=float("inf")), dict(scale=float("nan"))])
    size = abi.load_library().kvip_hip_chunk_attention_workspace_bytes
    assert size(0, 16, 4, 4, 4) == size(2, 129, 4, 4, 4) == size(2, 16, 0, 4, 4) == size(2, 16, 4, 0, 4) == 0
    assert size(2, 16, 4, 4, 0) == size(2, 16, 4, 4, (1 << 31) + 1) == size(2, 16, 4, (1 << 17) + 1, 4) == 0
    assert 1152 * 32 < size(1, 16, 65, 4, 1) < size(64, 16, 65, 4, 1 << 20) and size(64, 16, 65, 4, 1 << 20) > (1 << 20) * 1152
    # Few rows of the problem per request: tree attention's.
    tree = abi.load_library().kvip_hip_tree_attention_workspace_bytes
    assert size(1, 16, 32, 40, 1 << 20) == tree(1, 16, 32, 40) and size(1, 16, 33, 40, 1 << 20) > (1 << 20) * 1152
    assert size(2, 16, 64, 40, 1 << 20) == tree(2, 16, 64, 40) and size(2, 16, 65, 40, 1 << 20) > (1 << 20) * 1152


def test_norm_rotary_rejects_before_launch():
    tensor = dict(x=256, out=256, x_token=128, x_head=128, out_token=128, out_head=128, heads=1, norm=abi.NORM_RMS)

    def two(first, second=None):
        return (abi.NormTensor * 2)(abi.NormTensor(**first), abi.NormTensor(**(second or {})))

    good = dict(tensors=two(tensor, tensor), positions=256, frequencies=256, tokens=4, dim=128, rotary_dim=64,
                dtype=abi.DTYPE_BF16, epsilon=1e-6)
    rejects("kvip_hip_norm_rotary", abi.NormRotaryArgs, good, [
        dict(positions=0), dict(frequencies=0), dict(tokens=-1), dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=130),
        dict(dim=514), dict(dim=62), dict(dtype=abi.DTYPE_FP8_E4M3), dict(epsilon=-1.0), dict(epsilon=float("nan")),
        dict(tensors=two({})), dict(tensors=two({**tensor, "out": 0})), dict(tensors=two({**tensor, "heads": 0})),
        dict(tensors=two({**tensor, "norm": 3})), dict(tensors=two(tensor, {**tensor, "heads": 65537}))])
    codes, pages = dict(tensor, scales=256), dict(tensor, scales=256, out_token=128 * 128, out_head=128)
    good = dict(good, tensors=two(codes, pages), quantised=1, slots=256, num_blocks=2)
    rejects("kvip_hip_norm_rotary", abi.NormRotaryArgs, good, [
        dict(dim=64), dict(slots=0), dict(num_blocks=0), dict(tensors=two({**codes, "scales": 0}, pages)),
        dict(tensors=two({**codes, "out": 258}, pages)), dict(tensors=two({**codes, "out_head": 130}, pages)),
        dict(tensors=two(codes, {**pages, "heads": 2})), dict(tensors=two(codes, {**pages, "out_token": 128 * 64})),
        dict(tensors=two(codes, {**pages, "out_head": 64})), dict(tensors=two(codes, {**pages, "scales": 0}))])


def test_logits_and_histories_reject_before_launch():
    good = dict({f: 256 for f, _ in abi.LogitArgs._fields_[:16]}, logits_stride=100, probs_stride=100, batch=2, max_tokens=8,
                vocab=100, biases=3, dtype=abi.DTYPE_FP32, probs_dtype=abi.DTYPE_FP32)
    rejects("kvip_hip_process_logits", abi.LogitArgs, good, [
        dict(logits=0), dict(probs=0), dict(cu_seqlens=0), dict(workspace=0), dict(workspace=264), dict(seen=0), dict(counts=0),
        dict(tokens=0), dict(visible=0), dict(biases=-1), dict(biases=4097), dict(bias_tokens=0), dict(bias_values=0),
        dict(batch=0), dict(batch=1025), dict(max_tokens=0), dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(logits_stride=99),
        dict(probs_stride=99), dict(dtype=0), dict(probs_dtype=0),
        dict(max_tokens=1 << 20, vocab=1 << 20, logits_stride=1 << 20, probs_stride=1 << 20)])
    size = abi.load_library().kvip_hip_process_logits_workspace_bytes
    assert size(0, 100) == size(2, 0) == size(2, (1 << 20) + 1) == size(1 << 20, 1 << 20) == 0
    assert 0 < size(1, 1) < size(1, 4097) <= size(300, 4097)
    good = dict({f: 256 for f, _ in abi.HistoryArgs._fields_[:8]}, max_tokens=10, count=2, batch=2, vocab=100, token_stride=4)
    state = [dict(counts=0), dict(seen=0), dict(tokens=0), dict(batch=0), dict(batch=1025), dict(vocab=0), dict(vocab=(1 << 20) + 1)]
    rejects("kvip_hip_history_load", abi.HistoryArgs, good, state + [
        dict(requests=0), dict(cu_seqlens=0), dict(prompt_lens=0), dict(count=0), dict(count=1025), dict(max_tokens=-1),
        dict(max_tokens=1 << 31)])
    rejects("kvip_hip_history_append", abi.HistoryArgs, good, state + [dict(kept=0), dict(token_stride=0), dict(token_stride=65)])


def test_python_constructors_refuse():
    import torch

    chunk = dict(batch=2, heads=16, max_tokens=8, max_context=512, device="cuda:0")
    for bad in (dict(heads=0), dict(heads=129), dict(max_tokens=0), dict(max_context=0), dict(batch=0), dict(batch=1025),
                dict(max_rows=0), dict(output_dtype=torch.float16), dict(device="cpu")):
        with pytest.raises(ValueError):
            kvip_amd.ChunkAttention(torch, **{**chunk, **bad})
    for bad in (dict(batch=0), dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(device="cpu")):
        with pytest.raises(ValueError):
            kvip_amd.TokenHistory(torch, **{**dict(batch=2, vocab=100, device="cuda:0"), **bad})
    for bad in (dict(batch=0), dict(max_tokens=0), dict(vocab=0), dict(output_dtype=torch.float64), dict(device="cpu"),
                dict(max_tokens=1 << 20, vocab=1 << 20)):
        with pytest.raises(ValueError):
            kvip_amd.LogitProcessor(torch, **{**dict(batch=2, max_tokens=4, vocab=100, device="cuda:0"), **bad})

    class Turn:
        rotary_dim, device = 64, torch.device("cuda:0")

    for bad in (dict(dim=32), dict(dim=514), dict(dim=128, query_norm="mean"), dict(dim=128, epsilon=-1.0),
                dict(dim=128, epsilon=float("nan"))):
        with pytest.raises(ValueError):
            kvip_amd.NormRotary(torch, rotary=Turn(), **bad)
