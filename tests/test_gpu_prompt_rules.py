"""What the operators around a prompt chunk's layers (include/kvip_hip_prompt.h) owe their callers beyond ordinary inputs:
histories that only their bits speak for, tokens that tie, numbers at the ends of their range, calls that repeat
themselves, requests that claim the same rows. Values come from oracle/prompt.py or follow from the inputs."""
import math

import numpy as np
import pytest

import kvip_amd
from kvip_amd.runtime import abi
from oracle import prompt
from tests.test_gpu_draft import SCALE, device, dtype_of, host, say
from tests.test_gpu_prompt import Chunks, Sampling

pytestmark = pytest.mark.gpu


# --- logits ----------------------------------------------------------------------------------


@pytest.mark.parametrize("vocab,biases", [(60, 0), (700, 40), (9001, 300), (40000, 0)])
def test_counts_without_their_bit_are_not_read(torch_gpu, vocab, biases):
    """Counts of tokens that the request does not hold, next to tokens that it does, in the dense pass and in the lists; and a
    request that was cleared by its bits alone."""
    torch = torch_gpu
    say(f"case counts without bits vocab={vocab} biases={biases}")
    s = Sampling(torch, np.random.default_rng(vocab), [6, 1, 9, 2], vocab, "fp32", biases=biases)
    assert 0 < len(s.model.has[0]) < vocab
    s.history.seen[2] = 0
    s.model.wrote[2].clear()
    s.model.has[2].clear()
    counts, _ = s.model.arrays()
    for b, has in enumerate(s.model.has):
        others = np.setdiff1d(np.arange(vocab), list(has))
        counts[b, others] = 1 + others % 5
    s.history.counts.copy_(torch.from_numpy(counts))
    op = s.op()
    s.check(op())
    assert int(op.status.item()) == 0
