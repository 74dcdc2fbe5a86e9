"""The sliding attention's blocks of 256 rows, which batches of much work get: whole and in parts,
over both caches.  Small inputs get there in two ways: many sequences without a token (the launch is
laid out before lengths are known), or a large bound of the caches' lengths.  Tolerances are those of
test_gpu_sliding.py."""
import numpy as np
import pytest

import cache_ref as cref
import test_gpu_sliding as sl

pytestmark = pytest.mark.gpu


def wide(c, max_len=None):
    """Whether the call is laid out in blocks of 256 rows, whether it is cut, and into how many units."""
    T, heads, D = c["q"].shape
    n_kv, n_seq, window = c["k"].shape[1], len(c["off"]) - 1, c["max_window"]
    group = heads // n_kv
    max_len = c["max_len"] if max_len is None else max_len

    def steps(before, nodes):
        near = (c["reach"] or 1 << 31) + nodes + c["sinks"] + 128
        return (min(max_len + before, near) + 63) // 64 + 1

    most = own = mean = steps(window, window)
    if window > 64:
        own, mean = steps(window, 256 // group + 1), steps(window // 2, 256 // group + 1)
    row_blocks, units = -(-window * group // 256), n_seq * n_kv
    join = D // 64 + 1
    room = 256 * (own - join) // mean if own > join else 0
    return window * group > 128 and units >= 512 // (row_blocks * mean) + 1, \
        own * 2 >= most and units * row_blocks < room, \
        max(units, min(256 * own // mean // row_blocks, units * own // 4))


def whole(seed, sizes, lengths, *args, **kw):
    """With 600 empty sequences behind the first."""
    c = sl.case(seed, list(sizes) + [0] * 600, list(lengths) + [0] * 600, *args, **kw)
    assert wide(c)[:2] == (True, False)
    return sl.check(c)


def cut(c, max_len=10 ** 6):
    assert wide(c, max_len)[:2] == (True, True)
    return sl.check(c, max_len)


SHAPES = [(64, 2, 2), (128, 1, 5), (256, 1, 8)]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("reach,sinks", [(0, 0), (1, 0), (40, 3), (100, 0), (64, 130), (3000, 4)])
@pytest.mark.parametrize("D,n_kv,group", SHAPES)
def test_chunks(reach, sinks, q8, D, n_kv, group):
    kw = dict(reach=reach, sinks=sinks, q8=q8, chain=True)
    whole(D, [200, 65, 1, 0, 130], [0, 77, 300, 5, 64], n_kv, group, D, 16, pad=3, **kw)
    whole(reach, [300], [129], n_kv, group, D, 32, evict=True, **kw)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("reach,sinks", [(0, 0), (1, 2), (50, 0), (64, 70), (129, 4), (100000, 0)])
@pytest.mark.parametrize("D,n_kv,group", [(64, 2, 16), (128, 1, 11), (256, 1, 8)])
def test_trees(reach, sinks, q8, D, n_kv, group):
    kw = dict(reach=reach, sinks=sinks, q8=q8, evict=True)
    whole(D, [33, 64, 1, 17], [0, 500, 63, 129], n_kv, group, D, 16, branch=3, absent=True, pad=2, **kw)
    whole(sinks, [40], [200], n_kv, group, D, 64, chain=True, **kw)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D,n_kv,group", SHAPES)
def test_parts(q8, D, n_kv, group):
    """In parts: chunks, a tree, more than 64 sequences, a window that sees part of it."""
    cut(sl.case(D, [150, 70, 9], [2000, 0, 700], n_kv, group, D, 64, q8=q8, chain=True, pad=1))
    cut(sl.case(D, [64, 20], [1500, 65], n_kv, 8, D, 32, q8=q8, branch=2, absent=True))
    cut(sl.case(D, [0] * 33 + [90] + [0] * 31 + [3], [0] * 33 + [900] + [0] * 31 + [2000], 1, group, D,
                16, q8=q8, chain=True))
    cut(sl.case(D, [64] * 3, [1200, 3000, 0], n_kv, 8, D, 16, q8=q8, branch=2, reach=9000, sinks=4))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_few_parts_of_many_rows(q8, D):
    """So few that a workgroup joins several rows; parts of which some blocks see nothing."""
    for c in (sl.case(D, [150, 70, 1, 0, 149], [0, 900, 2000, 5, 64], 4, 2, D, 64, q8=q8, chain=True, pad=1),
              sl.case(D, [64, 20, 0, 33, 1], [700, 65, 9, 0, 1500], 4, 8, D, 32, q8=q8, branch=2, absent=True)):
        assert wide(c, 10 ** 6)[2] < 8 * 20
        cut(c)
    c = sl.case(D, [1000], [0], 2, 8, D, 16, q8=q8, chain=True)
    assert wide(c) == (True, True, 8)
    sl.check(c)


@pytest.mark.parametrize("q8", [False, True])
def test_more_units_than_the_host_counts_on(q8):
    """Two sequences of 10 and 15 steps, 25 units of one step, in turn by their last rows."""
    c = sl.case(4, [300, 270], [300, 640], 1, 8, 128, 32, q8=q8, chain=True, pad=2)
    assert wide(c, 10 ** 6)[2] == 25
    cut(c)


@pytest.mark.parametrize("q8", [False, True])
def test_parts_of_a_window(q8):
    sizes, lengths = [130, 200] * 5, [400, 0, 64, 3, 999, 250, 700, 65, 128, 1]
    c = sl.case(5, sizes, lengths, 4, 2, 64, 16, q8=q8, chain=True, reach=300, sinks=4, evict=True)
    cut(c, 999)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("reach", [0, 40])
def test_many_row_blocks(q8, reach):
    """Eight and more of a window, which are mapped to the chip in another order."""
    kw = dict(q8=q8, chain=True, reach=reach, pad=2)
    whole(7, [140, 0, 150, 7], [100, 3, 0, 513], 1, 16, 64, 16, **kw)
    c = sl.case(8, [300, 270], [129, 700], 1, 8, 128, 32, **kw)
    if reach == 0:
        cut(c)
    else:
        cut(sl.case(9, [300, 290, 0], [129, 17, 3], 4, 8, 128, 32, q8=q8, chain=True, reach=200, sinks=4), 129)


@pytest.mark.parametrize("group", [8, 16])
@pytest.mark.parametrize("reach,sinks", [(0, 0), (50, 3), (130, 70)])
def test_infinities_where_they_are_not_seen(group, reach, sinks):
    for sizes, chain in (([20], False), ([140], True)):
        c = sl.case(13, sizes + [0] * 600, [333] + [0] * 600, 1, group, 64, 16, reach=reach, sinks=sinks,
                    chain=chain, branch=2)
        assert wide(c)[0]
        used = set(c["pages"][c["pages"] >= 0].tolist())
        free = [p for p in range(c["kc"].shape[1]) if p not in used]
        for n in ("kc", "vc"):
            c[n][:, free] = np.nan
            c[n][:, c["pages"][0, 20], :, 13:] = np.inf
        for j in (333 - 48, 333 - 47, 333 - 100, 2, 69, 71):  # at borders of the windows
            c["vc"][0, c["pages"][0, j // 16], 0, j % 16, j % 64] = (np.inf, -np.inf, np.nan)[j % 3]
        c["v"][3, 0, 5], c["v"][5, 0, 60], c["v"][8, 0, 9] = np.inf, np.nan, -np.inf
        sl.check(c)


@pytest.mark.parametrize("reach", [0, 50])
def test_groups_of_nan_and_absent_pages(reach):
    for sizes, chain in (([20], False), ([140], True)):
        c = sl.case(17, sizes + [0] * 600, [333] + [0] * 600, 1, 8, 64, 16, reach=reach, sinks=3,
                    chain=chain, branch=2, q8=True)
        assert wide(c)[0]
        (k, ks), (v, vs) = c["codes"]
        for j in (333 - 48, 333 - 46, 1, 200):
            v[0, c["pages"][0, j // 16], 0, j % 16, :32] = 0
            vs[0, c["pages"][0, j // 16], 0, j % 16, 0] = np.nan
        gone = c["pages"][0, [3, 18]].copy()
        for n in (ks, vs):
            n[0, gone] = np.nan
        c["pages"][0, [3, 18]] = -1, 1 << 30
        c["kc"], c["vc"] = (cref.values(*x) for x in c["codes"])
        got = sl.check(c)
        assert np.isfinite(got[..., 32:]).all() and not np.isfinite(got[..., :32]).all()


@pytest.mark.parametrize("q8", [False, True])
def test_sharp_scores(q8):
    for sharp in (8.0, 60.0):
        whole(19, [70, 30], [500, 300], 1, 4, 128, 16, reach=400, sinks=4, q8=q8, sharp=sharp, chain=True)
