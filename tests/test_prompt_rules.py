"""What the Python side of the operators around a prompt chunk's layers owes its callers, without a GPU."""
import types

import torch

import kvip_amd
from kvip_amd.runtime import abi


def test_calls_of_a_history_do_not_mix(monkeypatch):
    """A call that another thread makes of the same object while the first is on its way into the library."""
    op = object.__new__(kvip_amd.TokenHistory)
    op.torch, op.device, op.batch, op.vocab = torch, torch.device("cpu"), 2, 100
    op.library = types.SimpleNamespace(kvip_hip_history_load="load", kvip_hip_history_append="append")
    op.counts, op.seen = torch.zeros((2, 100), dtype=torch.int32), torch.zeros((2, 4), dtype=torch.int32)
    op._args = abi.HistoryArgs(counts=op.counts.data_ptr(), seen=op.seen.data_ptr(), batch=2, vocab=100)
    prompt, out = torch.zeros(7, dtype=torch.int64), torch.zeros((2, 5), dtype=torch.int64)
    one, two = torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    calls, seen = {"load": lambda: op.load(one, prompt, two, one), "append": lambda: op.append(out, two)}, []

    def launch(t, device, entry, args, what):
        if not seen:
            seen.append(None)
            calls["append" if entry == "load" else "load"]()
        seen.append((entry, args.tokens, args.max_tokens if entry == "load" else args.token_stride, args.counts, args.vocab))

    monkeypatch.setattr(abi, "launch", launch)
    want = {("load", prompt.data_ptr(), 7, op.counts.data_ptr(), 100), ("append", out.data_ptr(), 5, op.counts.data_ptr(), 100)}
    for first in ("load", "append"):
        seen.clear()
        calls[first]()
        assert set(seen[1:]) == want, first
