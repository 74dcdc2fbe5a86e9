"""New lengths of a store beside the rows that it reads: in the gap between two tokens' rows."""
import numpy as np
import pytest
import torch

import test_gpu_window as w
from sager_amd import ops

pytestmark = pytest.mark.gpu
dev = w.dev


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("by_path", [False, True])
def test_between_rows(q8, by_path):
    layers, T, n_kv, D = 3, 7, 2, 64
    rng = np.random.default_rng(1)
    off, length = np.array([0, 3, 7], np.int32), np.array([5, 30], np.int32)
    pages = dev(np.arange(8, dtype=np.int32).reshape(2, 4))
    caches = []
    for _ in range(2):
        if q8:
            caches.append(ops.KvCacheQ8.empty(layers, 8, n_kv, 16, D, pages, dev(length)))
        else:
            caches.append(ops.KvCache(*(torch.zeros(layers, 8, n_kv, 16, D, dtype=torch.float16,
                                                    device="cuda") for _ in range(2)), pages, dev(length)))
    # a token's row: k, a gap of 8 values, v, a gap
    rows = dev(rng.normal(0, 1, (layers, T, 2 * (n_kv * D + 8))).astype(np.float16))
    k, v = (rows[..., a:a + n_kv * D].unflatten(2, (n_kv, D)) for a in (0, n_kv * D + 8))
    gap = rows[1, 2, n_kv * D + 2:n_kv * D + 6].view(torch.int32)
    path = dev(np.array([[0, 2, 0, 0], [0, 1, 3, 0]], np.int32)), dev(np.array([2, 3], np.int32))
    kept = rows.clone()
    for cache, out in zip(caches, (None, gap)):
        if by_path:
            got = cache.commit(k, v, dev(off), *path, length_out=out)
        else:
            got = cache.append(k, v, dev(off), max_window=4, length_out=out)
        assert got.tolist() == ([7, 33] if by_path else [8, 34])
    for n, t in caches[0]._tensors.items():
        assert torch.equal(t, caches[1]._tensors[n]), n
    rows[1, 2, n_kv * D + 2:n_kv * D + 6] = kept[1, 2, n_kv * D + 2:n_kv * D + 6]
    assert torch.equal(rows, kept)
