"""The sliding attention over batches of one sequence's chunk and the others' single tokens, and calls of
several sizes that share a workspace."""
import numpy as np
import pytest
import torch

import test_gpu_sliding as sl
import test_gpu_window as w
from sager_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("reach", [0, 40])
def test_a_chunk_among_single_tokens(q8, reach):
    """128 sequences with a bound of 4,096 tokens each, 64 heads."""
    rng = np.random.default_rng(7)
    lengths = [int(x) for x in rng.integers(0, 60, 128)]
    c = sl.case(reach, [1] * 50 + [150] + [1] * 77, lengths, 8, 8, 64, 16, reach=reach, sinks=3, q8=q8,
                chain=True, pad=2)
    c["max_window"] = 4096
    sl.check(c)


@pytest.mark.parametrize("q8", [False, True])
def test_windows_with_the_workspace_of_a_chunk(q8):
    """One object for a prompt's chunks, one for windows behind it, the chunks' workspace for both."""
    cs = [sl.case(5, [n], [3000], 2, 8, 128, 16, q8=q8, chain=True) for n in (700, 4)]
    made = [sl.make(c) for c in cs]
    big = ops.SlidingAttention(16, 2, 128, max_tokens=2000, max_window=2000, max_len=4000)
    for c, (op, cache) in zip(cs, made):
        want = w.run_attn(c, op, cache)
        got = op.forward(*(w.dev(c[n]) for n in ("q", "k", "v")), cache, w.dev(c["off"]),
                         scale=c["scale"], workspace=big.workspace)
        assert torch.equal(got, want)
