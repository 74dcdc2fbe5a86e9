"""Attention over a sliding window and the first tokens, over a 16-bit and a quantised cache, against
its plain form in 64 bits (a quantised value is code * scale there as here).  The tolerance is that of the tree attention's tests: the output's rounding, the
weights' (2^-11 each), fp32 sums, and what a score's fp32 error moves a weight by."""
import numpy as np
import pytest
import torch

import cache_ref as cref
import test_gpu_window as w
from sager_amd import ops

pytestmark = pytest.mark.gpu
dev = w.dev


def case(seed, sizes, lengths, n_kv, group, D, page, reach=0, sinks=0, q8=False, evict=False, **kw):
    c = w.attn_case(seed, sizes, lengths, n_kv, group, D, page, **kw)
    c.update(reach=reach, sinks=sinks, q8=q8)
    if q8:
        c["codes"] = [cref.quantise(c[n]) for n in ("kc", "vc")]
        c["kc"], c["vc"] = (cref.values(*x) for x in c["codes"])
    if evict:  # whole pages that nobody sees any more have gone to others
        for s, n in enumerate(lengths):
            for p in range((n + page - 1) // page):
                if p * page >= sinks and (p + 1) * page <= n - reach + 1:
                    c["pages"][s, p] = -1
    return c


def make(c, max_len=None, **kw):
    T, heads, D = c["q"].shape
    if c["q8"]:
        (k, ks), (v, vs) = c["codes"]
        cache = ops.KvCacheQ8(*(dev(x) for x in (k, v, ks, vs, c["pages"], c["length"])))
    else:
        cache = ops.KvCache(*(dev(c[n]) for n in ("kc", "vc", "pages", "length")))
    op = ops.SlidingAttention(heads, c["k"].shape[1], D, max_tokens=T, max_seqs=len(c["off"]) - 1,
                              max_window=c["max_window"],
                              max_len=c["max_len"] if max_len is None else max_len,
                              reach=c["reach"], sinks=c["sinks"], **kw)
    return op, cache


def plain(c, out):
    with np.errstate(over="ignore"):
        return cref.attention(c["q"], c["k"], c["v"], c["kc"][0], c["vc"][0], c["pages"], c["length"],
                              c["off"], c["parent"], c["scale"], c["page"], out, c["reach"],
                              c["sinks"], c["max_window"])


def check(c, max_len=None):
    T, heads, D = c["q"].shape
    op, cache = make(c, max_len)
    fill = torch.full((T, heads, D), 3.0, dtype=torch.float16, device="cuda")
    got = w.run_attn(c, op, cache, out=fill).cpu().numpy().astype(np.float64)
    want, spread = plain(c, np.full((T, heads, D), 3.0))
    tol = w.attn_tol(c, want, spread)
    np.testing.assert_array_equal(np.isfinite(got), np.isfinite(want))
    ok = np.isfinite(want)
    bad = np.abs(got[ok] - want[ok]) - tol[ok]
    assert (bad <= 0).all(), bad.max()
    assert (got[c["off"][-1]:] == 3.0).all()  # rows behind the last sequence
    return got


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n_kv,group", [(1, 1), (2, 8), (3, 3), (1, 16)])
@pytest.mark.parametrize("length", [0, 1, 17, 63, 64, 65, 500])
def test_lengths(D, n_kv, group, length, q8):
    """All of the cache: no window, no sinks."""
    check(case(length + D, [1], [length], n_kv, group, D, 16, q8=q8))
    check(case(length, [5, 2], [length, max(length - 3, 0)], n_kv, group, D, 32, branch=2, q8=q8))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("reach", [1, 2, 5, 63, 64, 65, 130, 100000, 2 ** 31 - 1])
@pytest.mark.parametrize("sinks", [0, 1, 4, 70, 310, 5000])
def test_windows_and_sinks(reach, sinks, q8):
    """One token, a chain, trees with absent nodes, caches shorter and longer than the window; pages
    that nobody sees are gone."""
    kw = dict(reach=reach, sinks=sinks, q8=q8, evict=True)
    check(case(reach + sinks, [1, 1, 1, 1], [0, 3, 300, 1000], 2, 2, 64, 16, **kw))
    check(case(sinks, [7, 1, 13], [299, 64, 2], 1, 3, 128, 32, branch=3, absent=True, pad=2, **kw))
    check(case(reach, [9], [700], 1, 4, 64, 16, chain=True, **kw))
    check(case(reach, [64], [200], 1, 1, 64, 64, branch=2, **kw))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("reach,sinks", [(0, 0), (1, 0), (40, 3), (100, 0), (64, 130), (3000, 4)])
@pytest.mark.parametrize("D,n_kv,group", [(64, 2, 1), (128, 1, 5), (256, 1, 8)])
def test_chunks(reach, sinks, q8, D, n_kv, group):
    """Chains longer than 64 tokens: ragged ones, behind caches and without one."""
    kw = dict(reach=reach, sinks=sinks, q8=q8, chain=True)
    check(case(D, [200, 65, 1, 0, 130], [0, 77, 300, 5, 64], n_kv, group, D, 16, pad=3, **kw))
    check(case(reach, [300], [129], n_kv, group, D, 32, evict=True, **kw))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("reach,sinks", [(0, 0), (700, 4), (2000, 90)])
def test_parts(D, q8, reach, sinks):
    """Caches long enough to be cut into parts, ragged ones, with and without a true bound."""
    c = case(D, [3, 1, 4], [4000, 65, 1100], 2, 4, D, 64, reach=reach, sinks=sinks, q8=q8, branch=2)
    got = check(c)
    np.testing.assert_allclose(check(c, max_len=10), got, rtol=0, atol=2e-3)
    check(case(D + 1, [16], [3000], 1, 8, D, 16, reach=reach, sinks=sinks, q8=q8, branch=2))


@pytest.mark.parametrize("q8", [False, True])
def test_many_sequences(q8):
    rng = np.random.default_rng(3)
    sizes = [int(x) for x in rng.integers(0, 3, 200)]
    lengths = [int(x) for x in rng.integers(0, 90, 200)]
    sizes[100], lengths[100], sizes[-1], lengths[-1] = 2, 3000, 1, 1500
    for reach, sinks in ((0, 0), (64, 4), (1000, 0)):
        check(case(7, sizes, lengths, 2, 1, 64, 16, reach=reach, sinks=sinks, q8=q8, chain=True, pad=2))


@pytest.mark.parametrize("q8", [False, True])
def test_absent_pages(q8):
    """Pages that are gone where they would be seen: their tokens are not attended to."""
    c = case(11, [2, 5], [500, 260], 2, 2, 128, 16, reach=300, sinks=40, q8=q8, branch=2)
    c["pages"][0, [1, 20, 30, 31]] = [-1, 1 << 30, -7, c["kc"].shape[1]]
    c["pages"][1, :] = -1
    check(c)


@pytest.mark.parametrize("group", [1, 8])
@pytest.mark.parametrize("reach,sinks", [(0, 0), (50, 3), (130, 70)])
def test_infinities_where_they_are_not_seen(group, reach, sinks):
    """In pages that are gone, behind the cache's end, in the window's other branches, before the
    sliding window of some rows and inside that of others: they reach those that see them only."""
    for sizes, chain in (([9], False), ([140], True)):
        c = case(13, sizes, [333], 1, group, 64, 16, reach=reach, sinks=sinks, chain=chain, branch=2,
                 evict=True)
        used = set(c["pages"][c["pages"] >= 0].tolist())
        free = [p for p in range(c["kc"].shape[1]) if p not in used]
        for n in ("kc", "vc"):
            c[n][:, free] = np.nan
            c[n][:, c["pages"][0, 20], :, 13:] = np.inf
        for j in (333 - 48, 333 - 47, 333 - 100, 2, 69, 71):  # at borders of the windows
            if c["pages"][0, j // 16] >= 0:
                c["vc"][0, c["pages"][0, j // 16], 0, j % 16, j % 64] = (np.inf, -np.inf, np.nan)[j % 3]
        c["v"][3, 0, 5], c["v"][5, 0, 60], c["v"][8, 0, 9] = np.inf, np.nan, -np.inf
        got = check(c)
        if not chain or reach == 50:
            assert np.isfinite(got).any() and not np.isfinite(got).all()


def test_a_group_of_nan_where_it_is_not_seen():
    """A quantised group that holds an infinity reads as NaN; rows that do not see it do not mind."""
    for sizes, chain in (([9], False), ([140], True)):
        c = case(17, sizes, [333], 1, 8, 64, 16, reach=50, sinks=3, chain=chain, branch=2, q8=True)
        (k, ks), (v, vs) = c["codes"]
        for j in (333 - 48, 333 - 46, 1, 200):
            v[0, c["pages"][0, j // 16], 0, j % 16, :32] = 0
            vs[0, c["pages"][0, j // 16], 0, j % 16, 0] = np.nan
        ks[0, c["pages"][0, 100 // 16], 0, 100 % 16, 1] = np.nan
        c["kc"], c["vc"] = (cref.values(*x) for x in c["codes"])
        got = check(c)
        assert np.isfinite(got[..., 32:]).all() and not np.isfinite(got[..., :32]).all()


@pytest.mark.parametrize("q8", [False, True])
def test_sharp_scores(q8):
    """Scores far apart, a reference point that moves often, scores of -infinity."""
    for sharp in (8.0, 60.0):
        check(case(19, [4, 1], [1500, 700], 1, 4, 128, 16, reach=900, sinks=4, q8=q8, sharp=sharp))
    c = case(23, [3], [100], 1, 2, 64, 16, reach=30, q8=q8, chain=True)
    c["q"][1, :, :] = 0
    c["k"][2, 0, 0], c["q"][2, :, 0] = -np.inf, 1
    check(c)


@pytest.mark.parametrize("q8", [False, True])
def test_layers_strides_and_streams(q8):
    """q, k and v as slices of one projection, a layer in the middle, a side stream."""
    c = case(29, [3, 6], [400, 90], 2, 4, 128, 16, reach=100, sinks=4, q8=q8, branch=2)
    op, cache = make(c)
    want = w.run_attn(c, op, cache)
    t = cache._tensors
    more = {n: torch.stack([torch.zeros_like(x[0]), x[0], torch.ones_like(x[0])])
            for n, x in t.items() if x.dim() == 5}
    big = type(cache)(*(more.get(n, x) for n, x in t.items()))
    T, heads, D = c["q"].shape
    qkv = torch.zeros(T, (heads + 4) * D + 8, dtype=torch.float16, device="cuda")
    q, k, v = (qkv[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in
               ((0, heads), (heads, heads + 2), (heads + 2, heads + 4)))
    for x, n in ((q, "q"), (k, "k"), (v, "v")):
        x.copy_(dev(c[n]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = op.forward(q, k, v, big, dev(c["off"]), dev(c["parent"]), layer=1, scale=c["scale"])
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("q8", [False, True])
def test_two_graphs_share_a_workspace(q8):
    """Replayed in turn on one stream, with eager calls and longer caches in between."""
    cs = [case(s, [5, 3], [2500, 900], 2, 4, 128, 16, reach=r, sinks=4, q8=q8, branch=2)
          for s, r in ((71, 0), (72, 0))]
    made = [make(c) for c in cs]
    op = made[0][0]
    args = [[dev(c[n]) for n in ("q", "k", "v")] for c in cs]
    rest = [(dev(c["off"]), dev(c["parent"])) for c in cs]
    outs, graphs = [torch.zeros_like(a[0]) for a in args], []
    for i in range(2):
        op.forward(*args[i], made[i][1], *rest[i], scale=cs[i]["scale"], out=outs[i])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            op.forward(*args[i], made[i][1], *rest[i], scale=cs[i]["scale"], out=outs[i])
        graphs.append(g)
    for turn in range(3):
        for i, g in enumerate(graphs):
            want = op.forward(*args[i], made[i][1], *rest[i], scale=cs[i]["scale"])
            outs[i].zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want)
            made[i][1].length.sub_(100 + turn)


def test_two_streams_at_once():
    cs = [case(s, [5, 3], [2500, 900], 2, 4, 128, 16, reach=600, sinks=4, q8=s % 2, branch=2)
          for s in (81, 82)]
    made = [make(c) for c in cs]
    want = [w.run_attn(c, *m) for c, m in zip(cs, made)]
    args = [[dev(c[n]) for n in ("q", "k", "v")] for c in cs]
    rest = [(dev(c["off"]), dev(c["parent"])) for c in cs]
    outs, streams = [torch.zeros_like(o) for o in want], [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                made[i][0].forward(*args[i], made[i][1], *rest[i], scale=cs[i]["scale"], out=outs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_past_two_gib_of_a_pool():
    """Pages past 2^31 values of a pool, 16-bit and quantised."""
    D, page, n_kv = 256, 256, 2
    n_pages = 2 ** 31 // (page * n_kv * D) + 6
    rng = np.random.default_rng(9)
    c = case(31, [2], [600], n_kv, 4, D, page, reach=300, sinks=2, chain=True)
    used = c["pages"][0, :3].copy()
    for q8 in (False, True):
        vals = [c[n][:, used] for n in ("kc", "vc")]
        codes = [cref.quantise(x) for x in vals]
        shape = (1, n_pages, n_kv, page, D)
        if q8:
            ts = [torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in range(2)]
            ts += [torch.zeros((*shape[:4], D // 32), dtype=torch.float16, device="cuda")
                   for _ in range(2)]
            src = [codes[0][0], codes[1][0], codes[0][1], codes[1][1]]
        else:
            ts = [torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in range(2)]
            src = vals
        at = torch.from_numpy(n_pages - 1 - rng.permutation(3)).cuda()
        for t, x in zip(ts, src):
            t[:, at] = dev(x)
        pages = -np.ones((1, 4), np.int32)
        pages[0, :3] = at.cpu().numpy()
        cache = (ops.KvCacheQ8 if q8 else ops.KvCache)(*ts, dev(pages), dev(c["length"]))
        op = ops.SlidingAttention(8, n_kv, D, max_tokens=2, max_window=2, max_len=600, reach=300,
                                  sinks=2)
        got = w.run_attn(c, op, cache).cpu().numpy().astype(np.float64)
        d = dict(c)
        if q8:
            for n, x in zip(("kc", "vc"), codes):
                d[n] = c[n].astype(np.float64)
                d[n][:, used] = cref.values(*x)
            k, v = cache.read(dev(np.zeros(1, np.int32)), dev(np.array([0, 600], np.int32)), 600)
            for t, x in ((k, d["kc"]), (v, d["vc"])):
                rows = np.concatenate([x[0, p].transpose(1, 0, 2) for p in used])[:600]
                assert (t[0].cpu().numpy() == rows.astype(np.float16)).all()
        want, spread = plain(d, np.zeros(c["q"].shape))
        assert (np.abs(got - want) <= w.attn_tol(c, want, spread)).all()
        del ts, cache


def test_refusals_of_the_python_layer():
    c = case(37, [2], [40], 1, 2, 64, 16, q8=True)
    op, cache = make(c)
    q, k, v = (dev(c[n]) for n in ("q", "k", "v"))
    off, par = dev(c["off"]), dev(c["parent"])
    tree = ops.TreeAttention(2, 1, 64, max_tokens=2, max_window=2, max_len=40)
    with pytest.raises(ops.SagerError, match="quantised"):
        tree.forward(q, k, v, cache, off, par)
    for bad in (dict(reach=-1), dict(sinks=-1)):
        with pytest.raises(ops.SagerError):
            ops.SlidingAttention(2, 1, 64, max_tokens=2, **bad)
    long = ops.SlidingAttention(2, 1, 64, max_tokens=100, max_window=100, max_len=40, reach=5)
    x, y = (torch.zeros(100, n, 64, dtype=torch.float16, device="cuda") for n in (2, 1))
    o = dev(np.array([0, 100], np.int32))
    assert long.forward(x, y, y, cache, o).shape == x.shape
    for call in (lambda: long.forward(x, y, y, cache, o, torch.zeros(100, dtype=torch.int32, device="cuda")),
                 lambda: op.forward(q, k, v, cache, off, par, layer=1),
                 lambda: op.forward(q.float(), k, v, cache, off, par),
                 lambda: op.forward(q, k[:1], v, cache, off, par),
                 lambda: op.forward(q, k, v, cache, off, par, workspace=op.workspace[:8].cpu()),
                 lambda: op.forward(x, y, y, cache, o), lambda: op.forward(q, k, v, cache, off, par, out=q)):
        with pytest.raises(ops.SagerError):
            call()
