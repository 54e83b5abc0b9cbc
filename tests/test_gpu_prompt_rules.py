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


@pytest.mark.parametrize("vocab,biases", [(20000, 4096), (140001, 2000), (3000, 600)])
def test_tokens_named_twice_repeat_themselves(torch_gpu, vocab, biases):
    """Lists whose entries meet in pairs, from other threads and other waves: every call gives the same bits."""
    torch = torch_gpu
    say(f"case named twice vocab={vocab} biases={biases}")
    rng = np.random.default_rng(biases)
    s = Sampling(torch, rng, [1] * 40, vocab, "fp32", biases=biases)
    s.numbers["temperature"][:] = 1.5
    for b in range(40):
        s.names[b, :biases // 2] = rng.permutation(vocab)[:biases // 2]
        s.names[b, biases // 2:] = np.roll(s.names[b, :biases // 2], 1 + 64 * b)
    op = s.op()
    first = op().clone()
    for _ in range(60):
        assert torch.equal(op(), first)
    s.check(first)


def test_one_token_of_many_named_twice(torch_gpu):
    """Lists of 4096 different tokens but for one pair, or one token named by drafts and biases alike."""
    torch = torch_gpu
    say("case one pair")
    rng = np.random.default_rng(21)
    s = Sampling(torch, rng, [1, 30], 30000, "fp32", biases=4096, masked=True)
    s.numbers["temperature"][:] = 0.9
    s.allowed[:, 0] |= 1
    for b in range(2):
        s.names[b] = rng.permutation(30000)[:4096]
    for pair in ((0, 1), (4095, 0), (511, 512), (100, 4000)):
        names = s.names.copy()
        s.names[:, pair[1]] = s.names[:, pair[0]]
        op = s.op()
        s.check(op())
        s.names = names
    s.names[:, 70], s.names[:, 3000] = s.tokens[s.cu[:-1] + [0, 5]], s.tokens[s.cu[:-1] + [0, 5]]
    op = s.op()
    s.check(op())
    assert int(op.status.item()) == 0
