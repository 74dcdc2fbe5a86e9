"""Rotary positions of so many tokens that a workgroup takes several rounds of a token's heads, and the
caches past 2^31 values of a pool."""
import numpy as np
import pytest
import torch

import cache_ref as cref
import test_gpu_rope as rp
from sager_amd import ops

pytestmark = pytest.mark.gpu
dev = rp.dev


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("nb", [False, True])
@pytest.mark.parametrize("T,H,K,D,rot", [(1100, 9, 2, 128, 128), (300, 16, 2, 256, 64), (600, 7, 3, 64, 22),
                                         (1030, 5, 5, 96, 50), (1200, 2, 1, 512, 512), (1500, 3, 4, 64, 64),
                                         (1025, 1, 1, 512, 300)])
def test_rope_of_many_tokens(T, H, K, D, rot, nb, dtype):
    rng = np.random.default_rng(T)
    pos = rng.integers(0, 200000, T).astype(np.int32)
    wq, wk = (rng.normal(1, 0.2, D).astype(np.float32) for _ in range(2))
    buf, t, q, k = rp.case(rng, T, H, K, D, dtype)
    x = [a.cpu().numpy() for a in (q, k)]
    ops.rope(q, k, ops.rope_frequencies(rot, 1e6), positions=dev(pos), interleaved=nb, mscale=1.25,
             q_norm=dev(wq), k_norm=dev(wk), eps=1e-5)
    for got, a, n in ((q, x[0], wq), (k, x[1], wk)):
        want, size = cref.rope(a, n, 1e-5, cref.turns(rot, 1e6), pos, nb, 1.25)
        rp.check(got, want, size, dtype)
    edge = t.cpu().numpy()
    assert (edge[:, 0] == buf[:, 0]).all() and (edge[:, -2:] == buf[:, -2:]).all()


@pytest.mark.parametrize("q8", [False, True])
def test_caches_past_two_gib_of_a_pool(q8):
    """Append and commit into the last pages of the last layer's pool, and reading them back."""
    D, page, n_kv, layers = 256, 256, 2, 2
    n_pages = 2 ** 31 // (page * n_kv * D) + 4
    rng = np.random.default_rng(3)
    pages, length = np.array([[n_pages - 1, n_pages - 3]], np.int32), np.array([250], np.int32)
    if q8:
        cache = ops.KvCacheQ8.empty(layers, n_pages, n_kv, page, D, dev(pages), dev(length))
    else:
        kv = [torch.zeros((layers, n_pages, n_kv, page, D), dtype=torch.float16, device="cuda")
              for _ in range(2)]
        cache = ops.KvCache(*kv, dev(pages), dev(length))
    k, v = (rng.normal(0, 1, (layers, 13, n_kv, D)).astype(np.float16) for _ in range(2))
    off = dev(np.array([0, 9], np.int32))
    new = cache.append(dev(k), dev(v), off)
    cache.length.copy_(new)
    off2 = dev(np.array([9, 13], np.int32))
    new = cache.commit(dev(k), dev(v), off2, dev(np.array([[0, 2, 3, 0]], np.int32)),
                       dev(np.array([3], np.int32)))
    assert new.tolist() == [262]
    rows = list(range(9)) + [9, 11, 12]
    at = [(pages[0, p // page], p % page) for p in range(250, 262)]
    for x, t, s in ((k, cache.k, "k_scale"), (v, cache.v, "v_scale")):
        got = torch.stack([t[:, p, :, i] for p, i in at], 1).cpu().numpy()
        if not q8:
            assert (got == x[:, rows]).all()
            continue
        code, scale = cref.quantise(x[:, rows])
        assert (got == code).all()
        sc = getattr(cache, s)
        assert (torch.stack([sc[:, p, :, i] for p, i in at], 1).cpu().numpy() == scale).all()
        assert int((t[:, :2] != 0).sum()) == 0
    if q8:
        back = cache.read(dev(np.array([250], np.int32)), dev(np.array([0, 12], np.int32)), 12)
        for got, x in zip(back, (k, v)):
            want = cref.values(*cref.quantise(x[:, rows])).astype(np.float16)
            assert (got.cpu().numpy() == want).all()
