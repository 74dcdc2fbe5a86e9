"""Attention whose parts of a cache are several steps of 64 keys long: both buffers of keys, the
reference point that moves after it was set, pages that are absent in the middle.  With max_len 0 a
call is not cut at all and every unit has all the steps; caches of 13,000 tokens are cut into parts
of three steps and more.  Then the commit of more layers than a thread copies at once.

Tolerances: p and the output are rounded to fp16 (u16 = 2^-11 each); a weight below fp16's least
number is off by up to 2^-33 of the largest; sums over n keys by n u32; a score by (D + 4) u32 of
scale * sum |q k| (not at all where only one product is not 0); its exponent by 2 u32 of itself for
the scale and the reference point, and as much for each time that the latter moves: two of them count,
since a move leaves what was there before at 2^-7."""
import numpy as np
import pytest
import torch

import test_gpu_window as w
import window_ref as ref
from sager_amd import load, ops

pytestmark = pytest.mark.gpu

U16, U32 = w.U16, w.U32
# window, group: blocks of 16 rows, of 32, of 256 with one and with two of them
FORMS = [(3, 4), (13, 3), (40, 5), (64, 8)]


def uncut_case(seed, window, group, D, lengths, n_kv=2, page=16, absent=True, sharp=1.0):
    return w.attn_case(seed, [window, max(1, window - 5)][:len(lengths)], lengths, n_kv, group, D,
                       page, branch=2, absent=absent, pad=2, sharp=sharp)


def run(c, max_len):
    T, heads, D = c["q"].shape
    n_kv, n_seq = c["k"].shape[1], len(c["off"]) - 1
    nbytes = load().sg_attn_tree_workspace_bytes(n_seq, c["max_window"], max_len, heads, n_kv, D)
    if max_len == 0:
        assert nbytes == 0  # not cut: every unit takes all of its sequence's steps
    else:
        steps = sum((n + 63) // 64 for n in c["length"]) * n_kv
        assert nbytes > 0 and steps >= 3 * (2 * n_seq * n_kv + 1024)  # three steps a part or more
    fill = torch.full((T, heads, D), 3.0, dtype=torch.float16, device="cuda")
    return w.run_attn(c, out=fill, max_len=max_len).cpu().numpy().astype(np.float64)


def plain(c):
    """ref.attention, all rows of a kv head at once: out, spread and the largest sum |q k|."""
    T, heads, D = c["q"].shape
    n_kv = c["k"].shape[1]
    G = heads // n_kv
    out, spread = np.full((T, heads, D), 3.0), np.zeros((T, heads, D))
    size = 0.0
    for s in range(len(c["off"]) - 1):
        a, up = int(c["off"][s]), ref.up_of(c["parent"], c["off"], s)
        n = len(up)
        at = np.arange(min(max(int(c["length"][s]), 0), c["pages"].shape[1] * c["page"]))
        pg = c["pages"][s, at // c["page"]]
        ok = (pg >= 0) & (pg < c["kc"].shape[1])
        pg, sl = pg[ok], (at % c["page"])[ok]
        see = np.zeros((n, n), bool)
        for i in range(n):
            see[i, ref.line_of(up, i)] = True
        seen = np.concatenate([np.tile(see.any(1)[:, None], (1, len(pg))), see], 1)
        for g in range(n_kv):
            K = np.concatenate([c["kc"][0, pg, g, sl], c["k"][a:a + n, g]]).astype(np.float64)
            V = np.concatenate([c["vc"][0, pg, g, sl], c["v"][a:a + n, g]]).astype(np.float64)
            q = c["q"][a:a + n, g * G:(g + 1) * G].astype(np.float64).reshape(n * G, D)
            x = np.where(np.repeat(seen, G, 0), q @ K.T * c["scale"], -np.inf)
            size = max(size, float((np.abs(q) @ np.abs(K).T).max()) * abs(c["scale"]))
            with np.errstate(invalid="ignore"):
                e = np.exp(x - x.max(1, keepdims=True))
                e = np.where(np.isnan(e), 0, e)
            tot = np.maximum(e.sum(1, keepdims=True), 1e-300)
            out[a:a + n, g * G:(g + 1) * G] = (e @ V / tot).reshape(n, G, D)
            spread[a:a + n, g * G:(g + 1) * G] = (e @ np.abs(V) / tot).reshape(n, G, D)
    return out, spread, size


def check(c, max_len=0, terms=None):
    got, (want, spread, size) = run(c, max_len), plain(c)
    D, n = c["q"].shape[2], int(c["length"].max()) + c["max_window"]
    score = (D + 4 if terms is None else terms) * U32 * size
    moved = 3 * 2 * U32 * size * 1.45
    tol = np.maximum(U16 * np.abs(want), 2.0 ** -25) + (U16 + n * U32 + 2 * score + moved) * spread
    tol += n * 2.0 ** -33 * float(np.abs(c["vc"].astype(np.float32)).max())
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
    assert (got[c["off"][-1]:] == 3.0).all()
    return got


@pytest.mark.parametrize("window,group", FORMS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("max_len", [0, 13000])
def test_attention_counts_every_key(D, window, group, max_len):
    """All scores 0 and each value a 1 in one column: the columns are the shares of the keys that
    have it, exact but for the division and the output's rounding.  A key lost or read twice changes
    a column by 1 in the keys of a column."""
    n_kv = 8 if max_len else 2
    lengths = [13000, 12990] if max_len else [1337, 409]
    page = 64 if max_len else 16
    rng = np.random.default_rng(D + window)
    sizes = [window, window - 1]
    off = ref.off_of(sizes)
    T = int(off[-1])
    parent = np.array(sum([ref.tree(rng, n, 3, True) for n in sizes], []), np.int32)
    per = [-(-n // page) for n in lengths]
    pages = -np.ones((2, max(per) + 1), np.int32)
    order = rng.permutation(sum(per))
    pages[0, :per[0]], pages[1, :per[1]] = order[:per[0]], order[per[0]:]
    kc = np.zeros((1, sum(per), n_kv, page, D), np.float16)
    vc = np.zeros_like(kc)
    v = np.zeros((T, n_kv, D), np.float16)
    col = lambda j, g: (7 * j + 3 * g + j // D) % D  # noqa: E731
    out = pages < -1
    for s in range(2):
        at = np.arange(lengths[s])
        for g in range(n_kv):
            vc[0, pages[s, at // page], g, at % page, col(at, g)] = 1
            i = np.arange(sizes[s])
            v[off[s] + i, g, col(lengths[s] + i, g)] = 1
        out[s, 3:per[s]:11] = True
    pages[out] = rng.choice([-1, sum(per), 1 << 30, -(1 << 31)], int(out.sum()))
    c = dict(q=np.zeros((T, n_kv * group, D), np.float16),
             k=rng.normal(0, 1, (T, n_kv, D)).astype(np.float16), v=v, kc=kc, vc=vc, pages=pages,
             length=np.array(lengths, np.int32), off=off, parent=parent, scale=1.0, page=page,
             max_window=window)
    got = run(c, max_len).reshape(T, n_kv, group, D)
    for s in range(2):
        up = ref.up_of(parent, off, s)
        at = np.arange(lengths[s])
        at = at[~out[s, at // page]]
        for g in range(n_kv):
            base = np.bincount(col(at, g), minlength=D)
            for i in range(sizes[s]):
                line = np.array(ref.line_of(up, i), int)
                n = base + np.bincount(col(lengths[s] + line, g), minlength=D)
                want = n / n.sum() if len(line) else n * 0.0
                err = np.abs(got[off[s] + i, g] - want)
                assert (err <= np.maximum((U16 + 4 * U32) * want, 2.0 ** -25)).all(), (s, g, i)


@pytest.mark.parametrize("window,group", FORMS)
@pytest.mark.parametrize("D,max_len", [(64, 0), (128, 0), (256, 0), (128, 13000)])
def test_attention_reference_point_moves(D, window, group, max_len):
    """Scores that grow along the cache by up to 32 (8) a step in some rows and fall, rest or grow
    slowly in others of the same tile: the sums so far are rescaled step after step."""
    lengths = [13000, 12990] if max_len else [700, 333]
    c = uncut_case(D + window, window, group, D, lengths, 8 if max_len else 2,
                   64 if max_len else 16)
    rng = np.random.default_rng(window)
    slope = 0.25 if not max_len else 1 / 16
    grow = lambda j: (j * slope).astype(np.float16)  # noqa: E731 (as fp16 rounds it)
    for n in ("q", "k", "kc"):
        c[n][:] = 0
    c["q"][..., 0] = rng.choice([2, 1, 0.5, -1, -0.25, 0], c["q"].shape[:2])
    for s in range(2):
        used = -(-int(c["length"][s]) // c["page"])
        j = np.arange(used * c["page"]).reshape(used, 1, c["page"])
        c["kc"][0, c["pages"][s, :used], :, :, 0] = grow(j)
        i = np.arange(c["off"][s], c["off"][s + 1])
        c["k"][i, :, 0] = rng.choice([0, 7, 300 * slope], (len(i), 1))
    c["scale"] = 1.0
    check(c, max_len, 0)


@pytest.mark.parametrize("window,group", FORMS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_of_sharp_scores(D, window, group):
    """Scores of a spread of 8, so that the reference point moves now and then; pages absent."""
    c = uncut_case(D - window, window, group, D, [905, 64], sharp=8.0)
    c["pages"][0, 5::9] = -1
    check(c)


@pytest.mark.parametrize("window,group", [(16, 1), (40, 1), (64, 4), (64, 8)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("length", [55, 64 * 5 + 60])
def test_attention_inf_and_nan_in_a_window_over_two_steps(D, window, group, length):
    """Infinities and NaN in values of the window on both sides of a step's end reach the nodes that
    see them and no others."""
    c = uncut_case(7, window, group, D, [length], 1, absent=False)
    base = check(c)
    up = ref.up_of(c["parent"], c["off"], 0)
    edge = 64 - length % 64  # the first node of the next step
    assert 0 < edge < window
    for bad in (np.inf, -np.inf, np.nan):
        d = dict(c, v=c["v"].copy())
        nodes = [edge - 1, edge, window - 1]
        for i, node in enumerate(nodes):
            d["v"][node, :, 5 + i] = bad
        got = run(d, 0)
        for i in range(window):
            hit = [5 + j for j, node in enumerate(nodes) if node in ref.line_of(up, i)]
            np.testing.assert_array_equal(np.delete(got[i], hit, 1), np.delete(base[i], hit, 1))
            same = np.isnan(got[i][:, hit]) if np.isnan(bad) else got[i][:, hit] == bad
            assert same.all(), (i, hit)


@pytest.mark.parametrize("layers", [7, 8, 9, 16, 17])
@pytest.mark.parametrize("D", [64, 256])
def test_commit_of_many_layers(layers, D):
    """Eight layers are one thread's, whole and in part; keys and values whose layers lie apart by
    something else than the cache's."""
    rng = np.random.default_rng(layers)
    n_kv, page, per, sizes, lengths = 3, 16, 3, [5, 2, 7], [14, 0, 31]
    off = ref.off_of(sizes)
    T, W = int(off[-1]) + 1, 7
    pages = rng.permutation(9).reshape(3, 3).astype(np.int32)
    big = lambda n: torch.from_numpy(  # noqa: E731
        rng.normal(0, 1, (layers, n, n_kv, page, D)).astype(np.float16)).cuda()
    kc, vc = big(9), big(9)
    buf = torch.from_numpy(rng.normal(0, 1, (layers, T + 3, 2, n_kv, D)).astype(np.float16)).cuda()
    k, v = buf[:, 1:T + 1, 0], buf[:, 1:T + 1, 1]
    path = -np.ones((3, W), np.int32)
    n_path = np.array([4, 1, 6], np.int32)
    path[0, :4], path[1, :1], path[2, :6] = [0, 2, 3, 4], 0, [0, 1, 2, 4, 5, 6]
    want_k, want_v = kc.cpu().numpy(), vc.cpu().numpy()
    hk, hv = k.cpu().numpy(), v.cpu().numpy()
    for s in range(3):
        for i in range(n_path[s]):
            p = lengths[s] + i
            want_k[:, pages[s, p // page], :, p % page] = hk[:, off[s] + path[s, i]]
            want_v[:, pages[s, p // page], :, p % page] = hv[:, off[s] + path[s, i]]
    i32 = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
    cache = ops.KvCache(kc, vc, i32(pages), i32(lengths))
    out = cache.commit(k, v, i32(off), i32(path), i32(n_path))
    np.testing.assert_array_equal(kc.cpu().numpy(), want_k)
    np.testing.assert_array_equal(vc.cpu().numpy(), want_v)
    np.testing.assert_array_equal(out.cpu().numpy(), np.array(lengths) + n_path)
