"""The quantised cache: what is written and what is read back, code by code and value by value (no
tolerances: the quantiser's rule has one answer, and a read value is rounded once)."""
import numpy as np
import pytest
import torch

import cache_ref as cref
import window_ref as ref
from sager_amd import ops

pytestmark = pytest.mark.gpu


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def make(rng, lengths, layers, n_kv, D, page, spare=2):
    """A cache with old codes in it, its table of pages in random order."""
    used = [(n + page - 1) // page for n in lengths]
    n_pages, per = sum(used) + spare, max(1, max(used))
    order, pages, at = rng.permutation(n_pages).astype(np.int32), -np.ones((len(used), per), np.int32), 0
    for i, u in enumerate(used):
        pages[i, :u] = order[at:at + u]
        at += u
    shape = (layers, n_pages, n_kv, page)
    k, v = (rng.integers(-127, 128, (*shape, D)).astype(np.int8) for _ in range(2))
    ks, vs = (rng.uniform(0.001, 0.1, (*shape, D // 32)).astype(np.float16) for _ in range(2))
    return k, v, ks, vs, pages


def put(c, pages, length, x, rows, kv):
    """Rows of x written as tokens length + i, into numpy copies."""
    code, scale = cref.quantise(x)
    S, (P, per) = c[0].shape[3], (c[0].shape[1], pages.shape[1])
    for s, r in enumerate(rows):
        for i, row in enumerate(r):
            p = length[s] + i
            if length[s] < 0 or p // S >= per or not 0 <= pages[s, p // S] < P:
                continue
            c[kv][:, pages[s, p // S], :, p % S] = code[:, row]
            c[kv + 2][:, pages[s, p // S], :, p % S] = scale[:, row]


def equal(cache, c):
    for got, want in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), c):
        got = got.cpu().numpy()
        if want.dtype == np.float16:  # (a NaN is a NaN)
            assert (np.isnan(got) == np.isnan(want)).all()
            assert (got[~np.isnan(got)] == want[~np.isnan(want)]).all()
        else:
            assert (got == want).all()


@pytest.mark.parametrize("layers", [1, 4, 7])
@pytest.mark.parametrize("sizes,lengths,n_kv,D,page", [
    ([4], [59], 2, 256, 64), ([1, 9, 0, 64], [0, 15, 3, 100], 5, 64, 16),
    ([3] * 40, list(range(40)), 1, 128, 32)])
def test_commit(layers, sizes, lengths, n_kv, D, page):
    rng = np.random.default_rng(D + layers)
    off, W = ref.off_of(sizes), max(sizes)
    T = int(off[-1]) + 2
    c = make(rng, [n + W for n in lengths], layers, n_kv, D, page)
    pages, length = c[4].copy(), np.array(lengths, np.int32)
    pages[0, -1], length[-1] = 99999, -1 if len(sizes) > 4 else length[-1]
    # k and v as slices of a projection's rows, every layer's
    kv = rng.normal(0, 1, (layers, T, 2 * n_kv * D + 5)).astype(np.float16)
    kv[..., ::37] *= 50
    buf = dev(kv)
    k, v = (buf[..., 1 + i * n_kv * D:1 + (i + 1) * n_kv * D].unflatten(2, (n_kv, D)) for i in (0, 1))
    path, n_path = -np.ones((len(sizes), W), np.int32), np.zeros(len(sizes), np.int32)
    rows = []
    for s, n in enumerate(sizes):
        r = sorted(rng.permutation(n)[:max(1, n // 2)].tolist()) if n else []
        path[s, :len(r)], n_path[s] = r, len(r)
        rows.append([int(off[s]) + i for i in r])
    cache = ops.KvCacheQ8(*(dev(x) for x in c[:4]), dev(pages), dev(length))
    got = cache.commit(k, v, dev(off), dev(path), dev(n_path))
    assert (got.cpu().numpy() == length + n_path).all()
    for i, t in enumerate((k, v)):
        put(c, pages, length, t.cpu().numpy(), rows, i)
    equal(cache, c[:4])


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("sizes,lengths,bound", [([1000, 3, 70, 0], [7, 0, 121, 5], None),
                                                 ([300, 20], [16, 40], 100)])
def test_append(q8, sizes, lengths, bound):
    """Chunks of any length into either cache; with a bound the rest is left out."""
    rng = np.random.default_rng(len(sizes))
    layers, n_kv, D, page = 2, 3, 128, 16
    off = ref.off_of(sizes)
    c = make(rng, [n + m for n, m in zip(lengths, sizes)], layers, n_kv, D, page)
    k, v = (rng.normal(0, 1, (layers, int(off[-1]) + 1, n_kv, D)).astype(np.float16) for _ in range(2))
    rows = [[int(off[s]) + i for i in range(min(n, bound or n))] for s, n in enumerate(sizes)]
    length = np.array(lengths, np.int32)
    if q8:
        cache = ops.KvCacheQ8(*(dev(x) for x in c), dev(length))
    else:
        half = [np.zeros(c[0].shape, np.float16) for _ in range(2)]
        cache = ops.KvCache(*(dev(x) for x in half), dev(c[4]), dev(length))
    got = cache.append(dev(k), dev(v), dev(off), max_window=bound)
    assert (got.cpu().numpy() == length + [len(r) for r in rows]).all()
    if q8:
        put(c, c[4], length, k, rows, 0)
        put(c, c[4], length, v, rows, 1)
        equal(cache, c[:4])
        return
    for i, x in enumerate((k, v)):
        for s, r in enumerate(rows):
            for j, row in enumerate(r):
                p = lengths[s] + j
                half[i][:, c[4][s, p // page], :, p % page] = x[:, row]
    assert (cache.k.cpu().numpy() == half[0]).all() and (cache.v.cpu().numpy() == half[1]).all()


def test_quantiser_at_its_edges():
    """Ties, subnormal scales, zeros, the largest numbers, infinities and NaN; every group of random
    16-bit patterns that is finite."""
    rng = np.random.default_rng(0)
    g = rng.integers(0, 1 << 16, (4000, 32)).astype(np.uint16)
    g[(g & 0x7C00) == 0x7C00] &= 0x83FF
    x = g.view(np.float16).copy()
    x[1000:2000] = (x[1000:2000].astype(np.float64) * 2.0 ** rng.integers(-30, 0, (1000, 1))).astype(np.float16)
    d = (rng.integers(1024, 2048, (1000, 1)) * 2.0 ** rng.integers(-20, -4, (1000, 1)))
    x[2000:3000] = (d * (rng.integers(-127, 127, (1000, 32)) + 0.5)).astype(np.float16)  # ties, or near
    x[2000:3000, 0] = (d[:, 0] * 127).astype(np.float16)
    x[3000:3100] = (rng.integers(-400, 400, (100, 32)) * 2.0 ** -24).astype(np.float16)
    x[3100], x[3101, 3:], x[3102] = 0, 0, -0.0
    x[3103, 0], x[3104, 31], x[3105, 7], x[3106, 16] = np.inf, -np.inf, np.nan, 65504
    x[3107:3200] = np.float16(65504) * np.sign(rng.normal(0, 1, (93, 32)))
    x[3200:] = (rng.normal(0, 1, (800, 32)) * 3).astype(np.float16)
    k = x.reshape(1, -1, 2, 64)
    T = k.shape[1]
    pages = np.arange((T + 15) // 16, dtype=np.int32)[None]
    cache = ops.KvCacheQ8.empty(1, pages.size, 2, 16, 64, dev(pages), dev(np.zeros(1, np.int32)))
    off = np.array([0, T], np.int32)
    cache.append(dev(k), dev(-k), dev(off))
    c = [np.zeros(cache.k.shape, np.int8), np.zeros(cache.k.shape, np.int8),
         np.zeros(cache.k_scale.shape, np.float16), np.zeros(cache.k_scale.shape, np.float16)]
    put(c, pages, [0], k, [range(T)], 0)
    put(c, pages, [0], -k, [range(T)], 1)
    equal(cache, c)
    got, _ = cache.read(dev(np.zeros(1, np.int32)), dev(off), T)
    with np.errstate(invalid="ignore"):
        want = cref.values(*cref.quantise(k)).astype(np.float16)
    got = got.cpu().numpy()
    odd = np.isnan(want)
    assert (np.isnan(got) == odd).all() and (got[~odd] == want[~odd]).all()
    assert np.isfinite(got).sum() == k.size - 3 * 32


@pytest.mark.parametrize("layers", [1, 3, 9])
@pytest.mark.parametrize("n_kv,D,page", [(2, 256, 64), (5, 64, 16), (1, 128, 32)])
def test_read(layers, n_kv, D, page):
    """Ranges from anywhere, past the table, on absent pages, of no tokens; strided outputs."""
    rng = np.random.default_rng(D + layers)
    lengths = [100, 3, 40, 64, 20]
    c = make(rng, lengths, layers, n_kv, D, page)
    c[4][2, 0], c[4][3, 1 % c[4].shape[1]] = -1, 1 << 30
    cache = ops.KvCacheQ8(*(dev(x) for x in c), dev(np.array(lengths, np.int32)))
    first, sizes = np.array([37, 0, 5, -2, 10 ** 9], np.int32), [61, 3, 0, 70, 2]
    off = ref.off_of(sizes)
    T = int(off[-1]) + 3
    got = cache.read(dev(first), dev(off), T)
    wide = torch.full((layers, T, 2 * n_kv * D + 3), 7.0, dtype=torch.float16, device="cuda")
    ko = wide[..., 1:1 + n_kv * D].unflatten(2, (n_kv, D))
    vo = torch.full((layers, T, n_kv, D), 7.0, dtype=torch.float16, device="cuda")
    cache.read(dev(first), dev(off), k_out=ko, v_out=vo)
    for i, (t, out) in enumerate(zip(got, (ko, vo))):
        val = cref.values(c[i], c[2 + i]).astype(np.float16)
        want = np.zeros((layers, T, n_kv, D), np.float16)
        for s, n in enumerate(sizes):
            for j in range(n):
                p = int(first[s]) + j
                if p >= 0 and p // page < c[4].shape[1] and 0 <= c[4][s, p // page] < c[0].shape[1]:
                    want[:, off[s] + j] = val[:, c[4][s, p // page], :, p % page]
        assert (t.cpu().numpy() == want).all()
        want[:, off[-1]:] = 7
        assert (out.cpu().numpy() == want).all()
    assert (wide[..., 0] == 7).all() and (wide[..., 1 + n_kv * D:] == 7).all()


def test_read_of_more_rows_than_a_page_table_of_sequences():
    """4,500 sequences of none, one or two rows."""
    rng = np.random.default_rng(2)
    n = 4500
    c = make(rng, [2] * n, 1, 1, 64, 16)
    sizes = rng.integers(0, 3, n).tolist()
    off = ref.off_of(sizes)
    cache = ops.KvCacheQ8(*(dev(x) for x in c), dev(np.full(n, 2, np.int32)))
    k, v = cache.read(dev(np.zeros(n, np.int32)), dev(off), int(off[-1]))
    for t, i in ((k, 0), (v, 1)):
        val = cref.values(c[i], c[2 + i]).astype(np.float16)
        want = np.concatenate([val[0, c[4][s, 0], 0, :m] for s, m in enumerate(sizes)])
        assert (t.cpu().numpy()[0, :, 0] == want).all()


def test_refusals_of_the_python_layer():
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    i32 = torch.int32
    code, scale = z(2, 4, 2, 16, 64, dt=torch.int8), z(2, 4, 2, 16, 2)
    pages, length = z(3, 4, dt=i32), z(3, dt=i32)
    for bad in ((code, code[:1], scale, scale, pages, length), (code.float(), code, scale, scale, pages, length),
                (code, code, scale[..., :1], scale, pages, length), (code, code, scale, scale.float(), pages, length),
                (code, code, scale, scale, pages, length[:2]), (code, code, scale, scale.cpu(), pages, length),
                (code[0], code[0], scale, scale, pages, length)):
        with pytest.raises(ops.SagerError):
            ops.KvCacheQ8(*bad)
    cache = ops.KvCacheQ8.empty(2, 4, 2, 16, 64, pages, length)
    with pytest.raises(AttributeError):
        cache.k_scale = scale
    k, off = z(2, 6, 2, 64), z(2, dt=i32)
    first = z(1, dt=i32)
    for call in (lambda: cache.append(k[:1], k, off), lambda: cache.append(k.float(), k, off),
                 lambda: cache.append(k, k, z(6, dt=i32)), lambda: cache.append(k, k, off, max_window=0),
                 lambda: cache.append(k[0], k[0], off),
                 lambda: cache.append(k, k, off, length_out=length[:1]),
                 lambda: cache.commit(k, k, off, z(1, 65, dt=i32), first),
                 lambda: cache.commit(k, k, off, z(2, 4, dt=i32), first),
                 lambda: cache.read(first, off), lambda: cache.read(first, off, 0),
                 lambda: cache.read(first, z(6, dt=i32), 4), lambda: cache.read(z(2, dt=i32), off, 4),
                 lambda: cache.read(first, off, k_out=k, v_out=k),
                 lambda: cache.read(first, off, k_out=k[0]),
                 lambda: cache.read(first.cpu(), off, 4),
                 lambda: cache.read(first, off, k_out=k, v_out=z(2, 5, 2, 64))):
        with pytest.raises(ops.SagerError):
            call()
