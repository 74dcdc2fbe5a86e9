"""Argument checks of the verify window's entry points, before any launch
(no GPU), and the plain forms that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import sager_amd
import window_ref as ref

P = ctypes.c_void_p
A = P(4096)
INVALID, GEOMETRY, UNSUPPORTED = 1, 4, 8


@pytest.fixture(scope="module")
def lib():
    return sager_amd.load()


def norm_args(**kw):
    a = dict(x=A, y=A, x_out=A, w=A, eps=1e-6, xn=A, xq=A, n=2048, rows=4)
    a.update(kw)
    return list(a.values()) + [None]


@pytest.mark.parametrize("f16", [False, True])
def test_norm_refusals(lib, f16):
    fn = lib.sg_add_rmsnorm_q8_k_f16 if f16 else lib.sg_add_rmsnorm_q8_k
    for kw, status in ((dict(x=None), INVALID), (dict(w=None), INVALID),
                       (dict(xn=None, xq=None), INVALID), (dict(x_out=None), INVALID),
                       (dict(y=None), INVALID), (dict(n=2000), GEOMETRY), (dict(n=0), GEOMETRY),
                       (dict(n=-256), GEOMETRY), (dict(rows=0), GEOMETRY), (dict(rows=-1), GEOMETRY),
                       (dict(n=16640), UNSUPPORTED), (dict(xq=P(4098)), INVALID),
                       (dict(x=P(4097)), INVALID), (dict(w=P(4098)), INVALID)):
        assert fn(*norm_args(**kw)) == status, kw
        assert b"sg_add_rmsnorm_q8_k" in lib.sg_last_error()


def cache(**kw):
    a = dict(k=4096, v=4096, pages=4096, length=4096, layer_stride=1 << 20, n_layers=2, n_pages=8,
             page_size=16, pages_per_seq=4, n_kv_heads=2, head_dim=128)
    a.update(kw)
    return sager_amd.KvCacheDesc(*a.values())


BAD_CACHES = [(dict(k=None), INVALID), (dict(pages=None), INVALID), (dict(length=None), INVALID),
              (dict(n_layers=0), GEOMETRY), (dict(n_pages=0), GEOMETRY),
              (dict(pages_per_seq=0), GEOMETRY), (dict(n_kv_heads=0), GEOMETRY),
              (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=512), UNSUPPORTED),
              (dict(page_size=8), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED),
              (dict(page_size=0), UNSUPPORTED), (dict(page_size=-16), UNSUPPORTED),
              (dict(page_size=1 << 30, pages_per_seq=4), UNSUPPORTED),
              (dict(k=4104), INVALID), (dict(layer_stride=4), INVALID)]


def attn_args(c, **kw):
    a = dict(q=A, k=A, v=A, qs=8 * 128, ks=256, vs=256, cache=ctypes.byref(c), layer=0, off=A,
             parent=A, out=A, ws=A, ws_bytes=1 << 40, n_seq=1, n_tokens=4, max_window=4, max_len=4000,
             n_heads=8, scale=0.1)
    a.update(kw)
    return list(a.values()) + [None]


def test_attention_refusals(lib):
    c = cache()
    for kw, status in ((dict(q=None), INVALID), (dict(v=None), INVALID), (dict(off=None), INVALID),
                       (dict(out=None), INVALID), (dict(cache=None), INVALID),
                       (dict(n_seq=0), GEOMETRY), (dict(n_tokens=0), GEOMETRY),
                       (dict(max_window=0), GEOMETRY), (dict(max_window=65), UNSUPPORTED),
                       (dict(layer=2), GEOMETRY), (dict(layer=-1), GEOMETRY),
                       (dict(max_len=-1), GEOMETRY), (dict(max_len=0x7FFFFFFF), UNSUPPORTED),
                       (dict(n_heads=7), GEOMETRY), (dict(n_heads=0), GEOMETRY),
                       (dict(qs=1023), GEOMETRY), (dict(ks=255), INVALID), (dict(ks=248), GEOMETRY),
                       (dict(vs=-256), GEOMETRY), (dict(k=P(4104)), INVALID),
                       (dict(out=P(4100)), INVALID), (dict(q=P(4097)), INVALID),
                       (dict(ws=None), INVALID), (dict(ws=P(4104)), INVALID),
                       (dict(ws_bytes=64), INVALID), (dict(n_seq=1 << 30), UNSUPPORTED)):
        assert lib.sg_attn_tree_f16(*attn_args(c, **kw)) == status, kw
        assert b"sg_attn_tree_f16" in lib.sg_last_error()
    for kw, status in BAD_CACHES:
        assert lib.sg_attn_tree_f16(*attn_args(cache(**kw))) == status, kw


def test_attention_workspace(lib):
    f = lib.sg_attn_tree_workspace_bytes
    assert f(0, 1, 1, 1, 1, 64) == 0 and f(1, 1, 1, 3, 2, 64) == 0
    assert f(1, 4, 100000, 16, 2, 256) > 0
    # what is enough for a batch is enough for a smaller one
    for max_len in (0, 100, 500, 100000):
        for args in ((4, max_len, 16, 2, 256), (1, max_len, 32, 8, 128), (64, max_len, 7, 7, 64)):
            for n in range(2, 400):
                assert f(n, *args) >= f(n - 1, *args)


def test_commit_refusals(lib):
    def args(c, **kw):
        a = dict(k=A, v=A, ks=256, vs=256, kl=4096, vl=4096, cache=ctypes.byref(c), off=A, path=A,
                 n_path=A, out=P(8192), n_seq=1, n_tokens=4, max_window=4)
        a.update(kw)
        return list(a.values()) + [None]
    c = cache()
    for kw, status in ((dict(k=None), INVALID), (dict(path=None), INVALID),
                       (dict(n_path=None), INVALID), (dict(off=None), INVALID),
                       (dict(cache=None), INVALID), (dict(out=A), INVALID), (dict(ks=255), GEOMETRY),
                       (dict(v=P(4097)), INVALID), (dict(n_seq=0), GEOMETRY),
                       (dict(max_window=65), UNSUPPORTED), (dict(n_seq=65536), UNSUPPORTED)):
        assert lib.sg_kv_commit_f16(*args(c, **kw)) == status, kw
    for kw, status in BAD_CACHES:
        assert lib.sg_kv_commit_f16(*args(cache(**kw))) == status, kw


def test_verify_refusals(lib):
    need = lib.sg_tree_verify_workspace_bytes(4, 1000, 2)
    assert lib.sg_tree_verify_workspace_bytes(4, 1000, 0) < need
    assert lib.sg_tree_verify_workspace_bytes(0, 1000, 0) == 0

    def args(**kw):
        a = dict(logits=A, tokens=A, off=A, parent=A, draft=A, temp=A, ua=A, us=A, path=A, n_path=A,
                 next=A, prob=A, ws=A, ws_bytes=need, n_seq=1, n_tokens=4, max_window=4, vocab=1000,
                 max_children=2)
        a.update(kw)
        return list(a.values()) + [None]
    for name in ("logits", "tokens", "off", "temp", "ua", "us", "path", "n_path", "next", "ws"):
        assert lib.sg_tree_verify(*args(**{name: None})) == INVALID, name
    for kw, status in ((dict(n_seq=0), GEOMETRY), (dict(n_tokens=0), GEOMETRY),
                       (dict(max_window=0), GEOMETRY), (dict(vocab=0), GEOMETRY),
                       (dict(max_children=0), GEOMETRY), (dict(max_window=65), UNSUPPORTED),
                       (dict(max_children=17), UNSUPPORTED), (dict(n_seq=65536), UNSUPPORTED),
                       (dict(vocab=(1 << 24) + 1), UNSUPPORTED), (dict(ws_bytes=need - 1), INVALID),
                       (dict(ws=P(4104)), INVALID)):
        assert lib.sg_tree_verify(*args(**kw)) == status, kw
        assert b"sg_tree_verify" in lib.sg_last_error()


# ---- the plain forms against what they stand for ------------------------------------

def test_plain_verify_keeps_the_target_distribution():
    """The token after the root has the target's probability, whatever the drafter proposes: summed
    over the drafter's tokens and a fine grid of both random numbers (two siblings, drawn from one
    distribution)."""
    rng = np.random.default_rng(0)
    V, N = 4, 60
    x = rng.normal(0, 1, (3, V)).astype(np.float32)
    p = ref.target(x[0], 1.0)
    q = rng.dirichlet(np.ones(V)).astype(np.float32)
    q = q / q.sum()
    grid = ((np.arange(N) + 0.5) / N).astype(np.float32)
    got = np.zeros(V)
    off, par = np.array([0, 3], np.int32), np.array([-1, 0, 0], np.int32)
    for a in range(V):
        for b in range(V):
            d = np.stack([q, q, q])
            for ua in grid[::3]:
                for ub in grid[::3]:
                    path, n, nxt, _ = ref.verify(x, np.array([0, a, b], np.int32), off, par, [1.0],
                                                 [0, ua, ub], [0.5], d)
                    w = q[a] * q[b] / (N // 3) ** 2
                    if n[0] == 2:
                        got[a if path[0, 1] == 1 else b] += w
                    else:
                        # the last draw over its own grid, from the rest that is left
                        for us in grid[::6]:
                            _, _, t, _ = ref.verify(x, np.array([0, a, b], np.int32), off, par,
                                                    [1.0], [0, ua, ub], [us], d)
                            got[t[0]] += w / len(grid[::6])
    # three grids of 20, 20 and 10 steps
    np.testing.assert_allclose(got, p, atol=0.06)
    assert abs(got.sum() - 1) < 1e-6


def test_plain_attention_of_one_key_is_its_value():
    q, k, v = (np.random.default_rng(1).normal(0, 1, (2, 1, 64)).astype(np.float16) for _ in range(3))
    c = np.zeros((1, 1, 16, 64), np.float16)
    out, _ = ref.attention(q, k, v, c, c, np.zeros((1, 1), np.int32), [0], np.array([0, 2]),
                           np.array([-1, 5]), 1.0, 16, np.zeros((2, 1, 64)))
    np.testing.assert_array_equal(out[0], v[0].astype(float))
    assert (out[1] == 0).all()


# ---- outputs over inputs -----------------------------------------------------------------

def test_attention_output_over_an_input(lib):
    c = cache()
    far = dict(q=P(1 << 30), k=P(2 << 30), v=P(3 << 30), ws=None)
    n = 4 * 8 * 128 * 2  # bytes of out, and of q
    for at in (1 << 30, (1 << 30) + n - 8, (1 << 30) - n + 8, 2 << 30, (2 << 30) + 4 * 512 - 8,
               3 << 30, (3 << 30) - 8):
        assert lib.sg_attn_tree_f16(*attn_args(c, **far, out=P(at))) == INVALID, at
        assert b"overlaps" in lib.sg_last_error()
    for at in ((1 << 30) + n, (1 << 30) - n, (2 << 30) + 4 * 512):  # beside: refused for its workspace
        assert lib.sg_attn_tree_f16(*attn_args(c, **far, out=P(at))) == INVALID, at
        assert b"workspace" in lib.sg_last_error()


def test_commit_lengths_over_the_cache_s(lib):
    c = cache()
    for out in (4096, 4096 + 4, 4096 - 4):
        args = [A, A, 256, 256, 4096, 4096, ctypes.byref(c), A, A, A, P(out), 2, 4, 4, None]
        assert lib.sg_kv_commit_f16(*args) == INVALID
        assert b"length_out" in lib.sg_last_error()


# ---- launches past what a grid holds ---------------------------------------------------

def test_launches_too_large(lib):
    for fn in (lib.sg_add_rmsnorm_q8_k_f16, lib.sg_add_rmsnorm_q8_k):
        assert fn(*norm_args(rows=1 << 22)) == UNSUPPORTED
    c = cache()
    for kw in (dict(n_seq=1 << 20, max_window=4, n_heads=8), dict(n_seq=1 << 21, max_window=1),
               dict(n_seq=1 << 15, max_window=64, n_heads=16, qs=2048),
               dict(n_seq=1 << 15, max_window=64, n_heads=8)):
        assert lib.sg_attn_tree_f16(*attn_args(c, **kw)) == UNSUPPORTED, kw
