"""Argument checks of rotary positions and the quantised cache, before any launch (no GPU), and the
rotary table against its plain form."""
import ctypes

import numpy as np
import pytest

import cache_ref as cref
import sager_amd

P = ctypes.c_void_p
INVALID, GEOMETRY, UNSUPPORTED = 1, 4, 8
ROOM = 1 << 30  # between buffers


@pytest.fixture(scope="module")
def lib():
    return sager_amd.load()


def at(i):
    return P(ROOM * i)


# ---- rotary positions -------------------------------------------------------------

def rope_args(**kw):
    a = dict(q=at(1), k=at(2), q_out=at(3), k_out=at(4), qs=1024, ks=256, qos=1024, kos=256,
             q_norm=at(5), k_norm=at(6), eps=1e-6, turns=at(7), mscale=1.0, positions=None,
             win_off=at(8), parent=at(9), length=at(10), n_tokens=4, n_seq=1, n_heads=8, n_kv=2,
             dim=128, rot=64, neighbours=0)
    a.update(kw)
    return list(a.values()) + [None]


@pytest.mark.parametrize("f16", [False, True])
def test_rope_refusals(lib, f16):
    fn = lib.sg_rope_f16 if f16 else lib.sg_rope
    for kw, status in ((dict(q=None), INVALID), (dict(q_out=None), INVALID), (dict(k=None), INVALID),
                       (dict(k_out=None), INVALID), (dict(turns=None), INVALID),
                       (dict(win_off=None), INVALID), (dict(length=None), INVALID),
                       (dict(n_tokens=0), GEOMETRY), (dict(n_seq=0), GEOMETRY),
                       (dict(n_heads=0), GEOMETRY), (dict(n_kv=-1), GEOMETRY),
                       (dict(dim=100), GEOMETRY), (dict(dim=0), GEOMETRY), (dict(rot=0), GEOMETRY),
                       (dict(rot=63), GEOMETRY), (dict(rot=130), GEOMETRY),
                       (dict(dim=520, qs=8000, ks=8000, qos=8000, kos=8000), UNSUPPORTED),
                       (dict(n_tokens=1 << 24), UNSUPPORTED), (dict(n_heads=1 << 21), UNSUPPORTED),
                       (dict(qs=1023), GEOMETRY), (dict(ks=255), GEOMETRY), (dict(qos=-1024), GEOMETRY),
                       (dict(kos=0), GEOMETRY), (dict(q=P(ROOM + 1)), INVALID),
                       (dict(k_norm=P(ROOM * 6 + 2)), INVALID), (dict(turns=P(ROOM * 7 + 4)), INVALID)):
        assert fn(*rope_args(**kw)) == status, kw
        assert b"sg_rope" in lib.sg_last_error()


@pytest.mark.parametrize("f16", [False, True])
def test_rope_outputs_over_what_is_read(lib, f16):
    fn, size = (lib.sg_rope_f16, 2) if f16 else (lib.sg_rope, 4)
    T, qw, kw = 4, 1024, 256
    sizes = dict(q=T * qw * size, k=T * kw * size, q_out=T * qw * size, k_out=T * kw * size,
                 q_norm=512, k_norm=512, turns=256, win_off=8, parent=16, length=4)
    place = {n: ROOM * (i + 1) for i, n in enumerate(sizes)}
    for out in ("q_out", "k_out"):
        for other in set(sizes) - {out}:
            spots = [place[other] + sizes[other] - 4, place[other] - sizes[out] + 4]
            if {out, other} not in ({"q_out", "q"}, {"k_out", "k"}):
                spots.append(place[other])
            for spot in spots:
                assert fn(*rope_args(**{out: P(spot)})) == INVALID, (out, other, spot)
                assert b"overlaps" in lib.sg_last_error()
    # positions instead of windows
    for out in ("q_out", "k_out"):
        assert fn(*rope_args(positions=at(20), **{out: P(ROOM * 20 + 12)})) == INVALID
    # q and k of one projection: another token's stride, q's rows over k's
    ld = 2048
    in_q, in_k = ROOM, ROOM + 1024 * size
    base = dict(q=P(in_q), k=P(in_k), q_out=P(in_q), k_out=P(in_k), qs=ld, ks=ld, qos=ld, kos=ld)
    for bad in (dict(qos=ld + 8), dict(k_out=P(in_k - size)), dict(k_out=P(in_k + ld * size)),
                dict(q_out=P(in_q + 8 * size)), dict(k=P(in_q + 1020 * size)),
                dict(q_out=P(in_q + (ld - 1000) * size))):
        assert fn(*rope_args(**{**base, **bad})) == INVALID, bad


@pytest.mark.parametrize("kind,code", [(None, 0), ("linear", 1), ("yarn", 2), ("by_turns", 3)])
@pytest.mark.parametrize("rot,base", [(64, 1e6), (2, 1e4), (128, 5e5), (50, 1e7)])
def test_rope_turns(lib, kind, code, rot, base):
    fast = 4.0 if kind == "by_turns" else 32.0
    got = np.zeros(rot // 2)
    assert lib.sg_rope_turns(got.ctypes.data, rot, base, code, 8.0, 8192.0, 1.0, fast) == 0
    np.testing.assert_allclose(got, cref.turns(rot, base, kind, 8.0, 8192.0, 1.0, fast), rtol=1e-13)
    assert (np.diff(got) < 0).all() or rot == 2


def test_rope_turns_refusals(lib):
    t = np.zeros(32)
    ok = [t.ctypes.data, 64, 1e4, 2, 4.0, 4096.0, 1.0, 32.0]
    assert lib.sg_rope_turns(*ok) == 0
    for i, v, status in ((0, None, INVALID), (1, 0, GEOMETRY), (1, 63, GEOMETRY), (1, -2, GEOMETRY),
                         (2, 1.0, INVALID), (2, float("nan"), INVALID), (3, 4, UNSUPPORTED),
                         (3, -1, UNSUPPORTED), (4, 0.0, INVALID), (4, float("inf"), INVALID),
                         (5, 0.0, INVALID), (6, 0.0, INVALID), (7, 1.0, INVALID),
                         (7, float("inf"), INVALID)):
        bad = list(ok)
        bad[i] = v
        assert lib.sg_rope_turns(*bad) == status, (i, v)


# ---- the quantised cache -------------------------------------------------------------

def cache(**kw):
    a = dict(k=ROOM, v=ROOM * 2, k_scale=ROOM * 3, v_scale=ROOM * 4, pages=ROOM * 5, length=ROOM * 6,
             layer_stride=1 << 20, n_layers=2, n_pages=8, page_size=16, pages_per_seq=4, n_kv_heads=2,
             head_dim=128)
    a.update(kw)
    return sager_amd.KvCacheQ8Desc(*a.values())


BAD_CACHES = [(dict(k=None), INVALID), (dict(v_scale=None), INVALID), (dict(pages=None), INVALID),
              (dict(length=None), INVALID), (dict(n_layers=0), GEOMETRY), (dict(n_pages=0), GEOMETRY),
              (dict(pages_per_seq=0), GEOMETRY), (dict(n_kv_heads=0), GEOMETRY),
              (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=512), UNSUPPORTED),
              (dict(page_size=8), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED),
              (dict(page_size=1 << 30, pages_per_seq=4), UNSUPPORTED), (dict(k=ROOM + 8), INVALID),
              (dict(k_scale=ROOM * 3 + 2), INVALID), (dict(layer_stride=(1 << 20) + 256), INVALID),
              (dict(layer_stride=8 * 2 * 16 * 128 - 512), GEOMETRY), (dict(layer_stride=-512), GEOMETRY)]


def store_args(c, by_path, **kw):
    a = dict(k=at(10), v=at(11), ks=256, vs=256, kl=4096, vl=4096, cache=ctypes.byref(c), off=at(12))
    if by_path:
        a.update(path=at(13), n_path=at(14))
    a.update(out=at(15), n_seq=2, n_tokens=4, max_window=4)
    a.update(kw)
    return list(a.values()) + [None]


@pytest.mark.parametrize("path", [True, False])
def test_store_refusals(lib, path):
    fn = lib.sg_kv_commit_q8 if path else lib.sg_kv_append_q8
    c = cache()
    cases = [(dict(k=None), INVALID), (dict(v=None), INVALID), (dict(off=None), INVALID),
             (dict(cache=None), INVALID), (dict(ks=255), GEOMETRY), (dict(vs=-256), GEOMETRY),
             (dict(v=P(4097)), INVALID), (dict(n_seq=0), GEOMETRY), (dict(n_tokens=0), GEOMETRY),
             (dict(max_window=0), GEOMETRY), (dict(n_seq=65536), UNSUPPORTED),
             (dict(max_window=0x7FFFFFFF), UNSUPPORTED)]
    if path:
        cases += [(dict(path=None), INVALID), (dict(n_path=None), INVALID),
                  (dict(max_window=65), UNSUPPORTED)]
    for kw, status in cases:
        assert fn(*store_args(c, path, **kw)) == status, kw
    for kw, status in BAD_CACHES:
        assert fn(*store_args(cache(**kw), path)) == status, kw
    # new lengths over what the launch still reads
    read = [(ROOM * 6, 2), (ROOM * 5, 8), (ROOM * 12, 3), (ROOM * 10, (4096 + 1024) // 2),
            (ROOM * 11, (4096 + 1024) // 2)] + ([(ROOM * 13, 8), (ROOM * 14, 2)] if path else [])
    for base, ints in read:
        for spot in (base, base + 4 * (ints - 1), base - 4):
            assert fn(*store_args(c, path, out=P(spot))) == INVALID, (base // ROOM, spot)
            assert b"length_out" in lib.sg_last_error()


def test_append_f16_refusals(lib):
    c = sager_amd.KvCacheDesc(ROOM, ROOM * 2, ROOM * 5, ROOM * 6, 1 << 20, 2, 8, 16, 4, 2, 128)
    fn = lib.sg_kv_append_f16
    for kw, status in ((dict(k=None), INVALID), (dict(off=None), INVALID), (dict(cache=None), INVALID),
                       (dict(ks=255), GEOMETRY), (dict(n_seq=65536), UNSUPPORTED),
                       (dict(max_window=0), GEOMETRY), (dict(max_window=0x7FFFFFFF), UNSUPPORTED),
                       (dict(out=P(ROOM * 6)), INVALID), (dict(out=P(ROOM * 12 + 4)), INVALID)):
        assert fn(*store_args(c, False, **kw)) == status, kw


def read_args(c, **kw):
    a = dict(cache=ctypes.byref(c), first=at(10), off=at(11), k=at(12), v=at(13), ks=256, vs=256,
             kl=1024, vl=1024, n_seq=2, n_rows=4)
    a.update(kw)
    return list(a.values()) + [None]


def test_read_refusals(lib):
    c = cache()
    for kw, status in ((dict(cache=None), INVALID), (dict(first=None), INVALID), (dict(off=None), INVALID),
                       (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(ks=255), GEOMETRY),
                       (dict(vs=0), GEOMETRY), (dict(kl=1023), GEOMETRY), (dict(vl=-1024), GEOMETRY),
                       (dict(n_seq=0), GEOMETRY), (dict(n_rows=0), GEOMETRY), (dict(k=P(4097)), INVALID),
                       (dict(n_rows=0x7FFFFFFF, kl=1 << 50, vl=1 << 50), UNSUPPORTED),
                       (dict(v=P(ROOM * 12 + 4094)), INVALID)):
        assert lib.sg_kv_read_q8(*read_args(c, **kw)) == status, kw
    for kw, status in BAD_CACHES:
        assert lib.sg_kv_read_q8(*read_args(cache(**kw))) == status, kw
    code = (1 << 20) + 8 * 2 * 16 * 128
    for i, n in ((1, code), (2, code), (3, code // 16), (4, code // 16), (5, 32), (10, 8), (11, 12)):
        for out in ("k", "v"):
            for spot in (ROOM * i, ROOM * i + n - 2, ROOM * i - 4094):
                assert lib.sg_kv_read_q8(*read_args(c, **{out: P(spot)})) == INVALID, (i, out)
                assert b"overlap" in lib.sg_last_error()


# ---- sliding attention -----------------------------------------------------------------

def attn_args(c, **kw):
    a = dict(q=at(20), k=at(21), v=at(22), qs=8 * 128, ks=256, vs=256, cache=ctypes.byref(c), layer=0,
             off=at(23), parent=at(24), out=at(25), ws=at(26), ws_bytes=1 << 40, n_seq=1, n_tokens=4,
             max_window=4, max_len=4000, n_heads=8, scale=0.1, reach=1000, sinks=4)
    a.update(kw)
    return list(a.values()) + [None]


def f16_cache(**kw):
    a = dict(k=ROOM, v=ROOM * 2, pages=ROOM * 5, length=ROOM * 6, layer_stride=1 << 20, n_layers=2,
             n_pages=8, page_size=16, pages_per_seq=4, n_kv_heads=2, head_dim=128)
    a.update(kw)
    return sager_amd.KvCacheDesc(*a.values())


@pytest.mark.parametrize("q8", [False, True])
def test_attention_refusals(lib, q8):
    fn = lib.sg_attn_sliding_q8 if q8 else lib.sg_attn_sliding_f16
    new = cache if q8 else f16_cache
    c = new()
    for kw, status in ((dict(q=None), INVALID), (dict(v=None), INVALID), (dict(off=None), INVALID),
                       (dict(out=None), INVALID), (dict(cache=None), INVALID), (dict(n_seq=0), GEOMETRY),
                       (dict(n_tokens=0), GEOMETRY), (dict(max_window=0), GEOMETRY),
                       (dict(max_window=65), UNSUPPORTED), (dict(layer=2), GEOMETRY),
                       (dict(layer=-1), GEOMETRY), (dict(max_len=-1), GEOMETRY),
                       (dict(max_len=0x7FFFFFFF), UNSUPPORTED), (dict(n_heads=7), GEOMETRY),
                       (dict(reach=-1), GEOMETRY), (dict(sinks=-1), GEOMETRY), (dict(qs=1023), GEOMETRY),
                       (dict(ks=255), INVALID), (dict(ks=248), GEOMETRY), (dict(vs=-256), GEOMETRY),
                       (dict(k=P(4104)), INVALID), (dict(out=P(4100)), INVALID), (dict(q=P(4097)), INVALID),
                       (dict(ws=None), INVALID), (dict(ws=P(4104)), INVALID), (dict(ws_bytes=64), INVALID),
                       (dict(n_seq=1 << 30), UNSUPPORTED),
                       (dict(parent=None, max_window=(1 << 24) + 1), UNSUPPORTED),
                       (dict(parent=None, max_window=1 << 24, n_heads=256, qs=256 * 128), UNSUPPORTED)):
        assert fn(*attn_args(c, **kw)) == status, kw
        assert b"sg_attn_sliding" in lib.sg_last_error()
    if q8:
        for kw, status in BAD_CACHES:
            assert fn(*attn_args(cache(**kw))) == status, kw
    # a window that ends past 32-bit positions
    far = new(page_size=1 << 20, pages_per_seq=2047, n_pages=1, layer_stride=1 << 40)
    assert fn(*attn_args(far)) != UNSUPPORTED
    assert fn(*attn_args(far, parent=None, max_window=1 << 24)) == UNSUPPORTED


@pytest.mark.parametrize("q8", [False, True])
def test_attention_output_over_what_is_read(lib, q8):
    fn = lib.sg_attn_sliding_q8 if q8 else lib.sg_attn_sliding_f16
    n_seq, T, W, heads, kv, D, n_pages, page, per = 3, 7, 4, 8, 2, 128, 9, 16, 4
    need = lib.sg_attn_sliding_workspace_bytes(n_seq, W, 4000, heads, kv, D, 1000, 4)
    assert need > 0
    layer, w = n_pages * kv * page * D, 1 if q8 else 2
    size = dict(q=T * heads * D * 2, k=T * kv * D * 2, v=T * kv * D * 2, kc=layer * w, vc=layer * w,
                pages=n_seq * per * 4, length=n_seq * 4, off=(n_seq + 1) * 4, parent=T * 4, ws=need)
    if q8:
        size.update(ks=layer // 16, vs=layer // 16)
    a, n_out = {n: ROOM * (i + 1) for i, n in enumerate(size)}, T * heads * D * 2
    geo = (layer, 2, n_pages, page, per, kv, D)
    if q8:  # (the second layer, the first one lies before the addresses)
        c = sager_amd.KvCacheQ8Desc(a["kc"] - layer, a["vc"] - layer, a["ks"] - layer // 16,
                                    a["vs"] - layer // 16, a["pages"], a["length"], *geo)
    else:
        c = sager_amd.KvCacheDesc(a["kc"] - 2 * layer, a["vc"] - 2 * layer, a["pages"], a["length"], *geo)

    def call(out, **kw):
        b = dict(a, **kw)
        return fn(P(b["q"]), P(b["k"]), P(b["v"]), heads * D, kv * D, kv * D, ctypes.byref(c), 1,
                  P(b["off"]), P(b["parent"]), P(out), P(b["ws"]), need, n_seq, T, W, 4000, heads, 0.1,
                  1000, 4, None)
    for other in size:
        for spot in (a[other], a[other] + (size[other] - 2) // 8 * 8, a[other] - n_out + 8):
            assert call(spot) == INVALID, (other, spot)
            assert b"overlaps" in lib.sg_last_error(), other


def test_attention_workspace(lib):
    f = lib.sg_attn_sliding_workspace_bytes
    assert f(0, 1, 1, 1, 1, 64, 0, 0) == 0 and f(1, 1, 1, 3, 2, 64, 0, 0) == 0
    assert f(1, 1, 1, 2, 2, 64, -1, 0) == 0 and f(1, 4, 100000, 16, 2, 256, 0, 0) > 0
    # what is enough for a batch is enough for a smaller one
    for max_len in (0, 100, 500, 100000):
        for reach, sinks in ((0, 0), (100, 4), (5000, 70)):
            for args in ((4, max_len, 16, 2, 256), (1, max_len, 32, 8, 128), (64, max_len, 7, 7, 64),
                         (1000, max_len, 8, 2, 128), (65, max_len, 4, 1, 256)):
                for n in range(2, 300):
                    assert f(n, *args, reach, sinks) >= f(n - 1, *args, reach, sinks)


@pytest.mark.parametrize("q8", [False, True])
def test_attention_token_strides(lib, q8):
    """A few tokens' rows are reached by 32-bit offsets."""
    fn = lib.sg_attn_sliding_q8 if q8 else lib.sg_attn_sliding_f16
    c = (cache if q8 else f16_cache)()
    for name in ("ks", "vs"):
        for stride in (1 << 27, 1 << 40):
            assert fn(*attn_args(c, n_tokens=1, max_window=1, **{name: stride})) == UNSUPPORTED
            assert b"stride" in lib.sg_last_error()
