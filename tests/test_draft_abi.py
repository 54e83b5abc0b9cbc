"""The C ABI and the Python checks of the drafted round's operators, without a GPU: exported symbols, struct
layouts, arguments rejected before any launch."""
import ctypes
import re
import subprocess
import textwrap

import pytest

import kvip_amd
from kvip_amd.runtime import abi
from tests.conftest import ROOT

HEADER = ROOT / "include" / "kvip_hip_draft.h"
STRUCTS = {
    "KvipPageTableArgs": abi.PageTableArgs,
    "KvipPagedRows": abi.PagedRows,
    "KvipRotaryTensor": abi.RotaryTensor,
    "KvipRotaryArgs": abi.RotaryArgs,
    "KvipRowStoreArgs": abi.RowStoreArgs,
    "KvipTreeAttnArgs": abi.TreeAttnArgs,
    "KvipVerifyArgs": abi.VerifyArgs,
}


def test_every_declared_symbol_is_exported():
    lib = abi.load_library()
    names = set(re.findall(r"^\s*uint(?:32|64)_t\s+(kvip_hip_\w+)\s*\(", HEADER.read_text(), re.M))
    assert names == set(abi.DRAFT_PROTOTYPES)
    assert all(hasattr(lib, name) for name in names)
    assert lib.kvip_hip_draft_abi_version() == abi.DRAFT_ABI_VERSION
    defines = dict(re.findall(r"#define KVIP_(\w+) (\d+)u?\b", HEADER.read_text()))
    for name in ("STATUS_NO_PAGE", "STATUS_BAD_LENGTH", "STATUS_BAD_TREE", "STATUS_BAD_PROBS", "DTYPE_FP16",
                 "DRAFT_MAX_NODES", "DRAFT_MAX_BATCH"):
        assert int(defines[name]) == getattr(abi, name), name


def test_ctypes_layout_matches_c(tmp_path):
    assert set(re.findall(r"typedef struct (\w+)", HEADER.read_text())) == set(STRUCTS)
    lines = []
    for cname, cls in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {field} %zu\\n", offsetof({cname}, {field}));' for field, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text(textwrap.dedent('#include <stddef.h>\n#include <stdio.h>\n#include "kvip_hip_draft.h"\nint main(void){\n'
                                   + "\n".join(lines) + "\nreturn 0;}\n"))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    layout = {(a, b): int(c) for a, b, c in (line.split() for line in out if line)}
    for cname, cls in STRUCTS.items():
        assert layout[(cname, "size")] == ctypes.sizeof(cls), cname
        for field, _ in cls._fields_:
            assert layout[(cname, field)] == getattr(cls, field).offset, (cname, field)


def rejects(entry, cls, good, cases):
    lib = abi.load_library()
    call = getattr(lib, entry)
    assert call(None, None) == abi.KVIP_ERR_INVALID
    for case in cases:
        args = cls(**{**good, **case})
        assert call(ctypes.byref(args), None) == abi.KVIP_ERR_INVALID, case


def test_page_tables_reject_before_launch():
    good = dict({f: 256 for f, _ in abi.PageTableArgs._fields_[:17]}, batch=2, max_blocks=4, num_blocks=8, max_tokens=16,
                path_stride=4, row_sets=1)
    state = [dict(block_table=0), dict(free_pages=0), dict(ticket=0), dict(batch=0), dict(batch=1025), dict(max_blocks=0),
             dict(max_blocks=(1 << 17) + 1), dict(num_blocks=0), dict(num_blocks=1 << 24)]
    rejects("kvip_hip_page_tables_extend", abi.PageTableArgs, good,
            state + [dict(counts=0), dict(visible=0), dict(max_tokens=0), dict(max_tokens=(1 << 20) + 1), dict(slots=0)])
    rejects("kvip_hip_page_tables_truncate", abi.PageTableArgs, good, state + [dict(targets=0)])
    rejects("kvip_hip_page_tables_move", abi.PageTableArgs, good,
            state + [dict(path=0), dict(path_stride=0), dict(rows=0), dict(row_sets=-1), dict(row_sets=65536)])


def test_rotary_and_store_reject_before_launch():
    tensor = abi.RotaryTensor(x=256, out=256, x_token=64, x_head=64, out_token=64, out_head=64, heads=1, dim=64)

    def two(first, second=None):
        return (abi.RotaryTensor * 2)(first, second or abi.RotaryTensor())

    good = dict(tensors=two(tensor), positions=256, frequencies=256, tokens=4, rotary_dim=64, dtype=abi.DTYPE_BF16)
    rejects("kvip_hip_rotary", abi.RotaryArgs, good, [
        dict(positions=0), dict(frequencies=0), dict(tokens=-1), dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=514),
        dict(rotary_dim=66), dict(dtype=abi.DTYPE_FP8_E4M3), dict(tensors=two(abi.RotaryTensor())),
        dict(tensors=two(tensor, abi.RotaryTensor(x=256, heads=1, dim=64))),
        dict(tensors=two(tensor, abi.RotaryTensor(x=256, out=256, heads=0, dim=64)))])
    good = dict(latent=256, rope=256, slots=256, positions=256, frequencies=256, kv_cache=256, latent_stride=512, rope_stride=64,
                kv_block_stride=128 * 656, tokens=4, row_stride=656, num_blocks=2, dtype=abi.DTYPE_BF16)
    rejects("kvip_hip_store_rows", abi.RowStoreArgs, good, [
        dict(latent=0), dict(slots=0), dict(frequencies=0), dict(kv_cache=264), dict(tokens=-1), dict(row_stride=640),
        dict(row_stride=660), dict(kv_block_stride=128 * 640), dict(kv_block_stride=128 * 656 + 8), dict(num_blocks=0),
        dict(dtype=0)])


def test_tree_attention_rejects_before_launch():
    good = dict({f: 256 for f, _ in abi.TreeAttnArgs._fields_[:10]}, kv_block_stride=128 * 656, row_stride=656, batch=2,
                heads=16, max_nodes=4, max_tokens=8, max_blocks=4, num_blocks=8, output_dtype=abi.DTYPE_BF16, scale=1.0)
    rejects("kvip_hip_tree_attention", abi.TreeAttnArgs, good, [
        dict(query=0), dict(query=264), dict(kv_cache=264), dict(output=260), dict(workspace=0), dict(workspace=264),
        dict(seq_lens=0), dict(cu_seqlens=0), dict(batch=0), dict(batch=1025), dict(heads=0), dict(heads=129),
        dict(max_nodes=0), dict(max_nodes=65), dict(max_tokens=0), dict(max_blocks=0), dict(max_blocks=(1 << 17) + 1),
        dict(num_blocks=0), dict(row_stride=640), dict(row_stride=664), dict(kv_block_stride=128 * 640),
        dict(output_dtype=abi.DTYPE_FP16), dict(row_stride=(1 << 24) + 16, kv_block_stride=1 << 32),
        dict(scale=float("inf")), dict(scale=float("nan")),
        dict(batch=1024, heads=128, max_nodes=64, max_blocks=1 << 17)])  # steps that 32 bits do not count
    size = abi.load_library().kvip_hip_tree_attention_workspace_bytes
    assert size(0, 16, 4, 4) == size(2, 129, 4, 4) == size(2, 16, 65, 4) == size(2, 16, 4, 0) == 0
    assert 0 < size(1, 16, 4, 1) < size(64, 16, 4, 1024)
    assert size(1024, 128, 64, 1 << 17) == 0


def test_verification_rejects_before_launch():
    good = dict({f: 256 for f, _ in abi.VerifyArgs._fields_[:12]}, parents=0, probs_stride=100, draft_stride=100, batch=2,
                max_nodes=4, max_tokens=8, vocab=100, dtype=abi.DTYPE_FP32)
    rejects("kvip_hip_verify_drafts", abi.VerifyArgs, good, [
        dict(probs=0), dict(tokens=0), dict(uniforms=0), dict(final_uniforms=0), dict(workspace=0), dict(workspace=260),
        dict(parents=256), dict(batch=0), dict(batch=1025), dict(max_nodes=0), dict(max_nodes=65), dict(max_tokens=0),
        dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(probs_stride=99), dict(draft_stride=99), dict(dtype=0)])
    size = abi.load_library().kvip_hip_verify_drafts_workspace_bytes
    assert size(0, 100) == size(2, 0) == 0 and 8 < size(1, 1) < size(3, 1) < size(3, 4097)


def test_python_constructors_refuse():
    import torch

    tables = dict(batch=2, max_context=512, num_blocks=8, max_tokens=16, device="cuda:0")
    for bad in (dict(batch=0), dict(batch=1025), dict(max_context=0), dict(num_blocks=0), dict(max_tokens=0), dict(device="cpu")):
        with pytest.raises(ValueError):
            kvip_amd.PageTables(torch, **{**tables, **bad})
    tree = dict(batch=2, heads=16, max_nodes=4, max_tokens=8, max_context=512, device="cuda:0")
    for bad in (dict(heads=129), dict(max_nodes=65), dict(max_tokens=0), dict(max_context=0), dict(batch=0),
                dict(output_dtype=torch.float16), dict(device="cpu")):
        with pytest.raises(ValueError):
            kvip_amd.TreeAttention(torch, **{**tree, **bad})
    verifier = dict(batch=2, max_nodes=4, vocab=100, device="cuda:0")
    for bad in (dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(max_nodes=65), dict(batch=0), dict(device="cpu")):
        with pytest.raises(ValueError):
            kvip_amd.DraftVerifier(torch, **{**verifier, **bad})
    for bad in (dict(rotary_dim=7), dict(rotary_dim=64, layout="pairs"), dict(rotary_dim=64, base=1.0), dict(rotary_dim=64)):
        with pytest.raises(ValueError):
            kvip_amd.Rotary(torch, device="cpu", **bad)
    with pytest.raises(ValueError):
        kvip_amd.KvRowStore(torch, kv_cache=torch.zeros(2, 128, 656, dtype=torch.uint8))
