"""The sliding attention over batches of one sequence's chunk and the others' single tokens."""
import numpy as np
import pytest

import test_gpu_sliding as sl

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
