"""The verify window's operators on the GPU against plain 64-bit forms.

Tolerances, from the roundings alone (u16 = 2^-11, u32 = 2^-24):
- norm: a sum of squares is at most 16 fp32 additions per lane and 12 over
  lanes and waves, so its square root is off by at most 14 u32, the division,
  root and two products by 4 more (18 u32 of the value, 24 taken); fp16
  buffers round once more (u16, or half of fp16's least step 2^-24).
- attention: p and the output are rounded to fp16 (u16 of sum p |v| and of
  the output), a weight below fp16's normal numbers is off by 2^-25 of a
  scale that is at least 2^8 above the row's largest weight's; the fp32 sums
  over n keys are off by at most n u32 of sum p |v|; a score is off by at most
  (D + 4) u32 of scale * sum |q k|.
- verification: fp64 within, prob rounds to fp32 once (u32 of it).
"""
import ctypes

import numpy as np
import pytest
import torch

import window_ref as ref
from sager_amd import ops

pytestmark = pytest.mark.gpu

U16, U32 = 2.0 ** -11, 2.0 ** -24


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


# ---- residual, norm, Q8_K -----------------------------------------------------

def check_norm(x, y, w, eps, dt, out="both", in_place=False):
    tx, ty, tw = dev(x), None if y is None else dev(y), dev(w)
    rows, n = x.shape
    xn = torch.full_like(tx, 7.0) if out != "q8" else None
    xq = ops.q8k_empty(rows, n) if out != "normed" else None
    keep = tx.clone()
    x_out = None if y is None else tx if in_place else torch.empty_like(tx)
    r, xn, xq = ops.add_rmsnorm_q8_k(tx, tw, eps, y=ty, x_out=x_out, xn=xn, xq=xq)
    r = r.cpu().numpy()
    with np.errstate(over="ignore"):
        want = x if y is None else (x.astype(np.float32) + y.astype(np.float32)).astype(dt)
    np.testing.assert_array_equal(r, want)
    if not in_place:
        assert torch.equal(tx, keep)
    f = want.astype(np.float64)
    n64 = f / np.sqrt((f * f).mean(1, keepdims=True) + np.float32(eps)) * w.astype(np.float64)
    if xn is not None:
        got = xn.cpu().numpy().astype(np.float64)
        tol = 24 * U32 * np.abs(n64)
        if dt == np.float16:
            tol = tol + np.maximum(U16 * np.abs(n64), 2.0 ** -25) * (1 + 24 * U32)
        assert (np.abs(got - n64) <= tol).all(), np.max(np.abs(got - n64) - tol)
    if xq is not None:
        base = xn
        if base is None:
            _, base, _ = ops.add_rmsnorm_q8_k(dev(want), tw, eps, xn=torch.empty_like(tx))
        assert torch.equal(xq, ops.quantize_q8_k(base))


@pytest.mark.parametrize("dt", [np.float16, np.float32])
@pytest.mark.parametrize("rows,n", [(1, 256), (1, 2048), (4, 2048), (5, 2304), (3, 5120), (2, 8448),
                                    (2, 16384), (131, 768), (517, 1280), (1100, 2048),
                                    (1025, 4096)])
def test_add_rmsnorm(dt, rows, n):
    rng = np.random.default_rng(rows * 7 + n)
    x = rng.normal(0, 2, (rows, n)).astype(dt)
    x[:, ::61] *= 20
    y = rng.normal(0, 1, (rows, n)).astype(dt)
    w = rng.normal(1, 0.3, n).astype(np.float32)
    check_norm(x, y, w, 1e-6, dt)
    check_norm(x, None, w, 1e-5, dt)
    check_norm(x, y, w, 1e-6, dt, out="q8", in_place=True)
    check_norm(x, y, w, 1e-6, dt, out="normed")


@pytest.mark.parametrize("dt", [np.float16, np.float32])
def test_add_rmsnorm_edge_values(dt):
    n = 512
    x = np.zeros((6, n), dt)
    x[1, 3] = 65504 if dt == np.float16 else 1e15   # one large value
    x[2] = np.array(6e-8, dt)                       # below fp16's normal numbers
    x[3] = 60000 if dt == np.float16 else 1e17      # a sum of squares past fp16
    x[4, ::2] = -1
    x[5, 0] = 1
    w = np.linspace(-2, 2, n).astype(np.float32)
    check_norm(x, None, w, 1e-6, dt)
    check_norm(x, None, w, 0.25, dt)


def test_add_rmsnorm_infinite_rows_stay_apart():
    """An infinite or NaN row (a sum past fp16's range) does not touch the others."""
    rng = np.random.default_rng(0)
    x = rng.normal(0, 1, (9, 768)).astype(np.float16)
    y = rng.normal(0, 1, (9, 768)).astype(np.float16)
    x[4, 100] = y[4, 100] = 65504
    x[7, 5] = np.nan
    w = np.ones(768, np.float32)
    r, xn, _ = ops.add_rmsnorm_q8_k(dev(x), dev(w), 1e-6, y=dev(y))
    assert torch.isinf(r[4, 100]) and torch.isnan(xn[4, 100]) and torch.isnan(xn[7]).all()
    keep = [i for i in range(9) if i not in (4, 7)]
    _, want, _ = ops.add_rmsnorm_q8_k(dev(x[keep]), dev(w), 1e-6, y=dev(y[keep]))
    assert torch.equal(xn[keep], want)


def test_add_rmsnorm_at_odd_addresses():
    """Rows whose buffers start at an odd element."""
    rng = np.random.default_rng(3)
    for dt in (torch.float16, torch.float32):
        rows, n = 3, 1024
        big = [torch.zeros(rows * n + 5, dtype=dt, device="cuda") for _ in range(4)]
        x, y, r, xn = (b[i + 1:i + 1 + rows * n].view(rows, n) for i, b in enumerate(big))
        x.copy_(dev(rng.normal(0, 1, (rows, n))))
        y.copy_(dev(rng.normal(0, 1, (rows, n))))
        w = torch.ones(n + 1, device="cuda")[1:]
        ops.add_rmsnorm_q8_k(x, w, 1e-6, y=y, x_out=r, xn=xn)
        a, b, _ = ops.add_rmsnorm_q8_k(x.clone(), w.clone(), 1e-6, y=y.clone())
        assert torch.equal(r, a) and torch.equal(xn, b)
        assert all((b[i + 1 + rows * n:] == 0).all() and (b[:i + 1] == 0).all()
                   for i, b in enumerate(big))


# ---- attention ------------------------------------------------------------------

def attn_case(seed, sizes, lengths, n_kv, group, D, page, branch=1, absent=False, pad=0, chain=False,
              scale=None, sharp=1.0):
    rng = np.random.default_rng(seed)
    off = ref.off_of(sizes)
    T = int(off[-1]) + pad
    parent = None if chain else np.array(
        sum([ref.tree(rng, n, branch, absent) for n in sizes], []) + [0] * pad, np.int32)
    per = max(1, max((n + page - 1) // page for n in lengths)) + 1
    used = [(n + page - 1) // page for n in lengths]
    n_pages = sum(used) + 2
    order = rng.permutation(n_pages)
    pages = -np.ones((len(sizes), per), np.int32)
    at = 0
    for i, u in enumerate(used):
        pages[i, :u] = order[at:at + u]
        at += u
    f16 = lambda *s: rng.normal(0, 1, s).astype(np.float16)  # noqa: E731
    return dict(q=f16(T, n_kv * group, D) * np.float16(sharp), k=f16(T, n_kv, D), v=f16(T, n_kv, D),
                kc=f16(1, n_pages, n_kv, page, D), vc=f16(1, n_pages, n_kv, page, D), pages=pages,
                length=np.array(lengths, np.int32), off=off, parent=parent,
                scale=D ** -0.5 if scale is None else scale, page=page,
                max_window=max(max(sizes), 1), max_len=max(lengths))


def attn_op(c, max_len=None, max_window=None, **kw):
    T, heads, D = c["q"].shape
    n_kv = c["k"].shape[1]
    cache = ops.KvCache(dev(c["kc"]), dev(c["vc"]), dev(c["pages"]), dev(c["length"]))
    op = ops.TreeAttention(heads, n_kv, D, max_tokens=T, max_seqs=len(c["off"]) - 1,
                           max_window=max_window or c["max_window"],
                           max_len=c["max_len"] if max_len is None else max_len, **kw)
    return op, cache


def run_attn(c, op=None, cache=None, out=None, **kw):
    if op is None:
        op, cache = attn_op(c, **kw)
    par = None if c["parent"] is None else dev(c["parent"])
    return op.forward(dev(c["q"]), dev(c["k"]), dev(c["v"]), cache, dev(c["off"]), par,
                      scale=c["scale"], out=out)


def attn_tol(c, want, spread):
    n = c["max_len"] + c["max_window"]
    D = c["q"].shape[2]
    score = (D + 4) * U32 * abs(c["scale"]) * D * float(np.nanmax(np.abs(c["q"].astype(float)))) * 5
    rel = U16 + n * U32 + score
    return np.maximum(U16 * np.abs(want), 2.0 ** -25) + rel * spread + n * 2.0 ** -33 * 6


def check_attn(c, **kw):
    T, heads, D = c["q"].shape
    fill = torch.full((T, heads, D), 3.0, dtype=torch.float16, device="cuda")
    got = run_attn(c, out=fill, **kw).cpu().numpy().astype(np.float64)
    want, spread = ref.attention(c["q"], c["k"], c["v"], c["kc"][0], c["vc"][0], c["pages"],
                                 c["length"], c["off"], c["parent"], c["scale"], c["page"],
                                 np.full((T, heads, D), 3.0),
                                 max_window=kw.get("max_window") or 64)
    tol = attn_tol(c, want, spread)
    np.testing.assert_array_equal(np.isfinite(got), np.isfinite(want))
    ok = np.isfinite(want)
    bad = np.abs(got[ok] - want[ok]) - tol[ok]
    assert (bad <= 0).all(), bad.max()
    assert (got[c["off"][-1]:] == 3.0).all()  # rows behind the last sequence
    return got


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n_kv,group", [(1, 1), (2, 8), (3, 3), (1, 16)])
@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 31, 33, 127, 500])
def test_attention_lengths(D, n_kv, group, length):
    check_attn(attn_case(length + D, [1], [length], n_kv, group, D, 16))
    check_attn(attn_case(length, [5, 2], [length, max(length - 3, 0)], n_kv, group, D, 32, branch=2))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 2, 3, 8, 17, 31, 32, 33, 63, 64])
def test_attention_windows(D, window):
    check_attn(attn_case(window, [window], [70], 2, 3, D, 16, branch=3))
    check_attn(attn_case(window, [window], [31], 1, 5, D, 64, chain=True))
    check_attn(attn_case(window, [window, 1, window], [0, 45, 96], 1, 2, D, 32, branch=4,
                         absent=True, pad=3))


@pytest.mark.parametrize("page", [16, 64, 1024])
def test_attention_ragged_batch(page):
    sizes, lengths = [3, 1, 7, 64, 2, 0, 5], [900, 0, 16, 333, 1500, 40, 64]
    check_attn(attn_case(page, sizes, lengths, 2, 4, 128, page, branch=2, absent=True, pad=4))


@pytest.mark.parametrize("D,length", [(64, 20011), (128, 9000), (256, 6001)])
def test_attention_split_over_long_caches(D, length):
    check_attn(attn_case(1, [4], [length], 1, 4, D, 64, branch=2))
    # longer than max_len promises, and shorter
    check_attn(attn_case(2, [4, 2], [length // 3, 50], 1, 2, D, 16, chain=True), max_len=700)
    check_attn(attn_case(3, [2], [300], 1, 2, D, 16, chain=True), max_len=100000)


def test_attention_rising_and_falling_scores():
    """Scores that grow along the cache move the reference point many times; scores that fall leave
    almost all weight on the first keys; very negative scores throughout."""
    for slope, shift in ((4.0, 0.0), (-4.0, 0.0), (0.02, -300.0)):
        c = attn_case(5, [3], [600], 1, 2, 64, 16, chain=True, scale=1.0)
        c["q"][:] = 0
        c["q"][:, :, 0], c["q"][:, :, 1] = 1, 1
        flat = c["kc"][0, c["pages"][0, :38], 0].reshape(-1, 64)
        flat[:, 0] = (np.arange(flat.shape[0]) * slope).astype(np.float16)
        flat[:, 1] = shift
        c["kc"][0, c["pages"][0, :38], 0] = flat.reshape(38, 16, 64)
        c["k"][:, :, 0] = np.array([[1.0], [600 * slope + 1], [-5]], np.float16)
        c["k"][:, :, 1] = shift
        want, spread = ref.attention(c["q"], c["k"], c["v"], c["kc"][0], c["vc"][0], c["pages"],
                                     c["length"], c["off"], c["parent"], 1.0, 16,
                                     np.zeros(c["q"].shape))
        got = run_attn(c).cpu().numpy().astype(np.float64)
        # a score of up to 2700 is off by (D + 4) u32 of it, and so is the exponent
        tol = U16 * np.abs(want) + (U16 + 700 * U32 + 68 * U32 * 2700) * spread + 1e-6
        assert (np.abs(got - want) <= tol).all()


def test_attention_absent_pages_and_lengths_out_of_range():
    c = attn_case(9, [2, 3, 1], [100, 64, 40], 2, 2, 128, 16, branch=2)
    c["kc"][0, -1] = np.nan  # a page nobody has
    c["vc"][0, -1] = np.nan
    c["pages"][0, 2] = -1
    c["pages"][0, 5] = 1 << 30
    c["pages"][1, 0] = c["kc"].shape[1]
    c["pages"][2, :] = -1            # nothing of it is left but its window
    check_attn(c)
    c["length"][1] = 1 << 30         # past the page table: the whole table
    c["length"][2] = -5
    c["pages"][1, 4:] = -1
    check_attn(c)


@pytest.mark.parametrize("D,group", [(64, 3), (128, 2), (256, 3), (128, 8), (64, 16), (128, 20),
                                     (256, 16), (256, 40), (64, 50)])
def test_attention_inf_and_nan_in_masked_places(D, group):
    """What a query does not see does not reach it: the slots behind the cache's end, the siblings in
    the tree, absent nodes.  (From 12 to 300 rows a kv head.)"""
    c = attn_case(11, [6], [37], 1, group, D, 16, branch=2)
    c["parent"][:] = [-1, 0, 0, 1, 2, 77]
    last = c["pages"][0, 2]
    c["kc"][0, last, :, 5:] = np.nan
    c["vc"][0, last, :, 5:] = np.inf
    base = check_attn(c)
    for bad in (np.inf, -np.inf, np.nan):
        d = {k: np.copy(v) if isinstance(v, np.ndarray) else v for k, v in c.items()}
        d["v"][2, :, 3] = bad            # node 2: seen by 2 and 4
        d["v"][5] = bad                  # absent
        d["k"][5] = bad
        got = run_attn(d).cpu().numpy().astype(np.float64)
        for node in (0, 1, 3):
            np.testing.assert_array_equal(got[node], base[node])
        for node in (2, 4):
            assert (np.isnan(got[node, :, 3]).all() if np.isnan(bad)
                    else (got[node, :, 3] == bad).all())
            np.testing.assert_array_equal(np.delete(got[node], 3, 1), np.delete(base[node], 3, 1))
        assert (got[5] == 0).all()
        d = {k: np.copy(v) if isinstance(v, np.ndarray) else v for k, v in c.items()}
        d["k"][2, 0, :] = np.nan         # a NaN score makes the rows that see it NaN, no others
        got = run_attn(d).cpu().numpy().astype(np.float64)
        for node in (0, 1, 3):
            np.testing.assert_array_equal(got[node], base[node])
        assert np.isnan(got[2]).all() and np.isnan(got[4]).all()


def test_attention_slices_layers_and_second_stream():
    """q, k and v as slices of one buffer, a layer of several, another stream."""
    c = attn_case(21, [3, 4], [90, 130], 2, 4, 128, 32, branch=2)
    T = c["q"].shape[0]
    want = run_attn(c)
    buf = torch.zeros((T, 12 * 128), dtype=torch.float16, device="cuda")
    q, k, v = buf.split([8 * 128, 2 * 128, 2 * 128], 1)
    q, k, v = q.view(T, 8, 128), k.view(T, 2, 128), v.view(T, 2, 128)
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        t.copy_(dev(c[n]))
    junk = torch.full((3, *c["kc"].shape[1:]), float("nan"), dtype=torch.float16, device="cuda")
    kc, vc = junk.clone(), junk.clone()
    kc[1], vc[1] = dev(c["kc"][0]), dev(c["vc"][0])
    cache = ops.KvCache(kc, vc, dev(c["pages"]), dev(c["length"]))
    op = ops.TreeAttention(8, 2, 128, max_tokens=T + 9, max_seqs=5, max_window=4, max_len=130)
    off, par = dev(c["off"]), dev(c["parent"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = op.forward(q, k, v, cache, off, par, layer=1, scale=c["scale"])
    side.synchronize()
    np.testing.assert_allclose(got.float().cpu().numpy(), want.float().cpu().numpy(), rtol=4e-3,
                               atol=2e-3)
    with pytest.raises(ops.SagerError):
        op.forward(q, k, v, cache, off, par, layer=3)


def test_attention_longer_window_than_promised():
    """Rows of a window past max_window are not seen: left as they were."""
    c = attn_case(31, [6], [50], 1, 2, 64, 16, chain=True)
    out = torch.full((6, 2, 64), 3.0, dtype=torch.float16, device="cuda")
    got = run_attn(c, max_window=4, out=out).cpu().numpy()
    c["max_window"] = 4
    want, _ = ref.attention(c["q"], c["k"], c["v"], c["kc"][0], c["vc"][0], c["pages"], c["length"],
                            c["off"], None, c["scale"], 16, np.full((6, 2, 64), 3.0), max_window=4)
    assert np.abs(got - want).max() < 0.02 and (got[4:] == 3).all()


def test_attention_offsets_past_32_bits():
    """A pool of more than 2^32 elements, its last pages used."""
    page, n_kv, D = 4096, 4, 128
    n_pages = (1 << 32) // (n_kv * page * D) + 3
    kc = torch.empty((1, n_pages, n_kv, page, D), dtype=torch.float16, device="cuda")
    vc = torch.empty_like(kc)
    ids = [n_pages - 1, n_pages - 3]
    c = attn_case(41, [3], [page + 200], n_kv, 2, D, page, branch=2)
    small = c["pages"][0, :2]
    for i, p in enumerate(ids):
        kc[0, p], vc[0, p] = dev(c["kc"][0, small[i]]), dev(c["vc"][0, small[i]])
    want = run_attn(c)
    op, _ = attn_op(c)
    pages = torch.tensor([ids + [-1]], dtype=torch.int32, device="cuda")
    cache = ops.KvCache(kc, vc, pages, dev(c["length"]))
    got = run_attn(c, op, cache)
    assert torch.equal(got, want)
    path = torch.tensor([[0, 2, -1]], dtype=torch.int32, device="cuda")
    n_path = torch.tensor([2], dtype=torch.int32, device="cuda")
    k = dev(c["k"])[None]
    cache.commit(k, k, dev(c["off"]), path, n_path)
    assert torch.equal(kc[0, ids[1], :, 200:202], k[0, [0, 2]].transpose(0, 1))


# ---- verification -----------------------------------------------------------------

def verify_case(seed, sizes, vocab, branch=1, absent=False, pad=0, chain=False, sampled=False,
                temps=(1.0, 0.7, 0.0, 1.4), peak=6.0):
    rng = np.random.default_rng(seed)
    off = ref.off_of(sizes)
    T = int(off[-1]) + pad
    parent = None if chain else np.array(
        sum([ref.tree(rng, n, branch, absent) for n in sizes], []) + [0] * pad, np.int32)
    x = rng.normal(0, 2, (T, vocab)).astype(np.float32)
    for r in x:
        r[rng.integers(0, vocab, 8)] += peak
    draft = None
    tokens = np.zeros(T, np.int32)
    q = np.zeros((T, vocab))
    for s in range(len(sizes)):
        for i in range(sizes[s]):
            p = i - 1 if parent is None else int(parent[off[s] + i])
            src = x[off[s] + (p if 0 <= p < i else 0)].astype(np.float64)
            g = src + rng.normal(0, 0.5, vocab)
            e = np.exp(g - g.max())
            q[off[s] + i] = e / e.sum()
            tokens[off[s] + i] = rng.choice(vocab, p=q[off[s] + i])
    if sampled:
        draft = q.astype(np.float32)
    return dict(logits=x, tokens=tokens, off=off, parent=parent, draft=draft,
                temp=np.array([temps[i % len(temps)] for i in range(len(sizes))], np.float32),
                u_acc=rng.random(T).astype(np.float32), u_smp=rng.random(len(sizes)).astype(np.float32))


def run_verify(c, max_children=16, max_window=None, op=None):
    T, V = c["logits"].shape
    W = max_window or max(1, int(np.diff(c["off"]).max()))
    op = op or ops.TreeVerify(V, max_tokens=T, max_seqs=len(c["off"]) - 1, max_window=W,
                              max_children=max_children if c["draft"] is not None else 0)
    prob = torch.full((T,), 5.0, device="cuda")
    got = op.forward(dev(c["logits"]), dev(c["tokens"]), dev(c["off"]),
                     None if c["parent"] is None else dev(c["parent"]), dev(c["temp"]),
                     dev(c["u_acc"]), dev(c["u_smp"]),
                     None if c["draft"] is None else dev(c["draft"]), prob=prob)
    return [t.cpu().numpy() for t in got]


def check_verify(c, max_children=16, max_window=None):
    T = len(c["tokens"])
    W = max_window or max(1, int(np.diff(c["off"]).max()))
    got = run_verify(c, max_children, W)
    want = ref.verify(c["logits"], c["tokens"], c["off"], c["parent"], c["temp"], c["u_acc"],
                      c["u_smp"], c["draft"], max_children, W, prob=np.full(T, 5.0))
    for g, w in zip(got[:3], want[:3]):
        np.testing.assert_array_equal(g, w)
    assert (np.abs(got[3] - want[3]) <= U32 * want[3] + 1e-12).all()
    return got


@pytest.mark.parametrize("vocab", [1, 2, 7, 255, 2047, 2048, 2049, 5003, 50257])
@pytest.mark.parametrize("sampled", [False, True])
def test_verify_vocabularies(vocab, sampled):
    for seed in range(3):
        check_verify(verify_case(seed, [4, 1, 3], vocab, branch=2, sampled=sampled))
        check_verify(verify_case(seed, [3], vocab, chain=True, sampled=sampled))


@pytest.mark.parametrize("window", [1, 2, 5, 31, 63, 64])
@pytest.mark.parametrize("sampled", [False, True])
def test_verify_windows(window, sampled):
    for branch in (1, 2, 5):
        check_verify(verify_case(window, [window, 0, max(1, window // 2), window], 613, branch=branch,
                                 absent=branch > 1, pad=2, sampled=sampled))


@pytest.mark.parametrize("sampled", [False, True])
def test_verify_many_sequences(sampled):
    """Enough draws that every way down the tree is taken."""
    c = verify_case(5, [1 + i % 9 for i in range(150)], 97, branch=3, sampled=sampled, peak=3.0)
    path, n_path, _, _ = check_verify(c)
    assert n_path.min() == 1 and n_path.max() >= 4


@pytest.mark.parametrize("sampled", [False, True])
def test_verify_large_vocabulary(sampled):
    check_verify(verify_case(6, [4], 248320, chain=True, sampled=sampled))
    # a vocabulary of more chunks than the last kernel has threads
    check_verify(verify_case(7, [2], 2048 * 1024 + 4097, chain=True, sampled=sampled))


def test_verify_acceptance_is_the_target_distribution():
    """Over all values of the random numbers the token after the root has the target's probability:
    the operator's formulas against what they are for (exact sums over a grid of u)."""
    V, N = 3, 512
    rng = np.random.default_rng(8)
    x = rng.normal(0, 1, (2, V)).astype(np.float32)
    p = ref.target(x[0], 1.0)
    q = np.array([0.2, 0.5, 0.3], np.float32)
    count = np.zeros(V)
    u = ((np.arange(N) + 0.5) / N).astype(np.float32)
    for tok in range(V):
        c = dict(logits=np.tile(x, (N * 8, 1)), tokens=np.tile(np.array([0, tok], np.int32), N * 8),
                 off=(2 * np.arange(N * 8 + 1)).astype(np.int32), parent=None,
                 draft=np.tile(q, (2 * N * 8, 1)), temp=np.ones(N * 8, np.float32),
                 u_acc=np.repeat(np.repeat(u, 8), 2), u_smp=np.tile((np.arange(8) + .5) / 8, N))
        c["u_smp"] = c["u_smp"].astype(np.float32)
        path, n_path, nxt, _ = run_verify(c, 1)
        after = np.where(n_path == 2, tok, nxt)
        count += q[tok] * np.bincount(after, minlength=V) / (N * 8)
    # 512 steps of u_accept and 8 of u_sample: a border is off by up to one step of each
    np.testing.assert_allclose(count, p, atol=3 / N + 1 / 8)


def test_verify_edge_logits_and_numbers():
    inf, nan = np.inf, np.nan
    x = np.zeros((12, 6), np.float32)
    x[0] = [-inf, 2, -inf, 2, -inf, -inf]   # ties: the lowest index at temperature 0
    x[1] = -inf                             # nothing left
    x[2] = [nan, 1, nan, 0, -inf, -1]
    x[3] = [inf, 0, inf, 3, -inf, nan]      # infinite logits share the mass
    x[4] = [1e30, -1e30, 0, 0, 0, 0]
    x[5] = nan
    off = np.arange(13, dtype=np.int32)
    for t in (0.0, 1.0, 0.01, 50.0, -1.0, nan, inf, 1e-30):
        for u in (0.0, 0.3, 0.5, 0.99, 1 - 2.0 ** -24):
            check_verify(dict(logits=x, tokens=np.zeros(12, np.int32), off=off, parent=None,
                              draft=None, temp=np.full(12, t, np.float32),
                              u_acc=np.full(12, u, np.float32), u_smp=np.full(12, u, np.float32)))
    # the same, one after the other in windows, with tokens out of range and equal siblings
    par = np.array([-1, 0, 0, 0, 1, 1, -1, 0, 0, 1, 1, 2], np.int32)
    tok = np.array([9, 1, 1, 3, -4, 6, 0, 2, 2, 1 << 30, 0, 0], np.int32)
    rng = np.random.default_rng(2)
    for t in (0.0, 1.0, 3.0):
        for sampled in (False, True):
            for _ in range(6):
                d = rng.dirichlet(np.ones(6), 12).astype(np.float32)
                check_verify(dict(logits=x, tokens=tok, off=np.array([0, 6, 12], np.int32),
                                  parent=par, draft=d if sampled else None,
                                  temp=np.full(2, t, np.float32),
                                  u_acc=rng.random(12).astype(np.float32),
                                  u_smp=rng.random(2).astype(np.float32)))


def test_verify_children_past_max_children():
    c = verify_case(12, [12, 9], 301, branch=5, sampled=True)
    for most in (1, 2, 4):
        check_verify(c, max_children=most)


def test_verify_drafter_is_the_target():
    """q = p: every draft is accepted, whatever the random number."""
    x = np.random.default_rng(1).normal(0, 2, (5, 700)).astype(np.float32)
    q = np.stack([ref.target(x[max(i - 1, 0)], 1.0) for i in range(5)])
    tok = q.argmax(1).astype(np.int32)
    c = dict(logits=x, tokens=tok, off=np.array([0, 5], np.int32), parent=None,
             draft=(q * (1 - 2.0 ** -20)).astype(np.float32), temp=np.ones(1, np.float32),
             u_acc=np.full(5, 1 - 2.0 ** -24, np.float32), u_smp=np.full(1, 0.5, np.float32))
    path, n_path, _, prob = check_verify(c, 1)
    assert n_path[0] == 5 and (prob == 1).all()


# ---- commit -------------------------------------------------------------------------

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page,layers,n_kv", [(16, 1, 1), (16, 3, 5), (64, 2, 2)])
def test_commit(D, page, layers, n_kv):
    rng = np.random.default_rng(D + page)
    sizes, lengths = [4, 1, 0, 9, 5], [15, 0, 3, 2 * page - 1, 4 * page - 2]
    off = ref.off_of(sizes)
    T, n, W, per = int(off[-1]) + 2, len(sizes), 9, 4
    pages = rng.permutation(n * per).reshape(n, per).astype(np.int32)
    shape = (layers, n * per + 1, n_kv, page, D)
    f16 = lambda *s: rng.normal(0, 1, s).astype(np.float16)  # noqa: E731
    kc, vc, k, v = f16(*shape), f16(*shape), f16(layers, T, n_kv, D), f16(layers, T, n_kv, D)
    path = -np.ones((n, W), np.int32)
    n_path = np.array([3, 1, 2, 9, 5], np.int32)
    path[0, :3], path[1, 0], path[2, :2] = [0, 1, 3], 0, [0, 1]  # (window 2 is empty)
    path[3] = np.arange(9)
    path[4, :5] = [0, 2, 7, -3, 4]                               # two nodes out of range
    pages[3, 2] = 10 ** 6                                        # an absent page
    cache = ops.KvCache(dev(kc), dev(vc), dev(pages), dev(np.array(lengths, np.int32)))
    # tokens of one buffer with the values and other things between them
    kv = torch.zeros((layers, T, 2 * n_kv * D + 8), dtype=torch.float16, device="cuda")
    tk = kv[:, :, :n_kv * D].view(layers, T, n_kv, D)
    tv = kv[:, :, n_kv * D:2 * n_kv * D].view(layers, T, n_kv, D)
    tk.copy_(dev(k))
    tv.copy_(dev(v))
    length = cache.commit(tk, tv, dev(off), dev(path), dev(n_path))
    for s in range(n):
        for i in range(n_path[s]):
            p = lengths[s] + i
            if 0 <= path[s, i] < sizes[s] and p // page < per and pages[s, p // page] < shape[1]:
                kc[:, pages[s, p // page], :, p % page] = k[:, off[s] + path[s, i]]
                vc[:, pages[s, p // page], :, p % page] = v[:, off[s] + path[s, i]]
    np.testing.assert_array_equal(cache.k.cpu().numpy(), kc)
    np.testing.assert_array_equal(cache.v.cpu().numpy(), vc)
    np.testing.assert_array_equal(length.cpu().numpy(), np.array(lengths) + n_path)
    np.testing.assert_array_equal(cache.length.cpu().numpy(), lengths)


def test_commit_counts_out_of_range():
    kc = torch.zeros((1, 4, 1, 16, 64), dtype=torch.float16, device="cuda")
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = ops.KvCache(kc, kc.clone(), i32([0, 1], [2, 3]), i32(-3, 5))
    k = torch.ones((1, 4, 1, 64), dtype=torch.float16, device="cuda")
    length = cache.commit(k, k, i32(0, 2, 4), i32([0, 1], [0, 1]), i32(1 << 30, -9))
    assert (kc == 0).all() and length.tolist() == [-1, 5]


# ---- together ---------------------------------------------------------------------

class Step:
    """One step of a session's window: norm, projections, attention, output projection, norm, head,
    verification, commit - the library's calls in the order a session makes them."""

    H, HEADS, KV, D, V = 512, 4, 2, 64, 1031

    def __init__(self, seed, sizes, lengths, layers=2):
        from sager_amd.synth import q4k_random_np
        rng = np.random.default_rng(seed)
        H, A = self.H, (self.HEADS + 2 * self.KV) * self.D
        q4 = lambda rows, k: dev(q4k_random_np(rng, rows * k // 256))  # noqa: E731
        self.w_qkv = [q4(A, H) for _ in range(layers)]
        self.w_o = [q4(H, self.HEADS * self.D) for _ in range(layers)]
        self.w_head = q4(self.V, H)
        self.norm = [dev(rng.normal(1, 0.1, H).astype(np.float32)) for _ in range(2 * layers + 1)]
        self.layers, self.sizes = layers, sizes
        self.off = ref.off_of(sizes)
        T = self.T = int(self.off[-1])
        c = attn_case(seed, sizes, lengths, self.KV, self.HEADS // self.KV, self.D, 16, branch=2)
        self.parent = dev(c["parent"])
        self.win_off = dev(self.off)
        pages = np.arange(len(sizes) * 8, dtype=np.int32).reshape(len(sizes), 8)
        kc = rng.normal(0, 1, (layers, pages.size, self.KV, 16, self.D)).astype(np.float16)
        self.cache = ops.KvCache(dev(kc), dev(kc[::-1]), dev(pages), dev(np.array(lengths, np.int32)))
        W = self.W = max(sizes)
        self.attn = ops.TreeAttention(self.HEADS, self.KV, self.D, T, len(sizes), W, max(lengths))
        self.verify = ops.TreeVerify(self.V, T, len(sizes), W)
        self.x0 = dev(rng.normal(0, 1, (T, H)).astype(np.float16))
        self.tokens = dev(rng.integers(0, self.V, T).astype(np.int32))
        self.temp = dev(np.array([0.0, 1.0, 0.7, 0.0][:len(sizes)], np.float32))
        self.u = dev(rng.random(T).astype(np.float32))
        self.us = dev(rng.random(len(sizes)).astype(np.float32))
        self.qkv = torch.zeros((layers, T, A), dtype=torch.float16, device="cuda")
        self.o = torch.zeros((T, self.HEADS, self.D), dtype=torch.float16, device="cuda")
        self.x = torch.zeros_like(self.x0)
        self.xn = torch.zeros_like(self.x0)
        self.xq = ops.q8k_empty(T, H)
        self.logits = torch.zeros((T, self.V), device="cuda")
        self.out = (torch.zeros((len(sizes), W), dtype=torch.int32, device="cuda"),
                    torch.zeros(len(sizes), dtype=torch.int32, device="cuda"),
                    torch.zeros(len(sizes), dtype=torch.int32, device="cuda"),
                    torch.zeros(T, device="cuda"))
        self.length = torch.zeros(len(sizes), dtype=torch.int32, device="cuda")

    def run(self):
        H, T, HD, KD = self.H, self.T, self.HEADS * self.D, self.KV * self.D
        self.x.copy_(self.x0)
        y = None
        for i in range(self.layers):
            ops.add_rmsnorm_q8_k(self.x, self.norm[2 * i], 1e-6, y=y,
                                 x_out=None if y is None else self.x, xn=self.xn, xq=self.xq)
            ops.gemv_q4_k_q8_f16out_batched(self.w_qkv[i], self.xq, HD + 2 * KD, H, T,
                                            y=self.qkv[i])
            q, k, v = self.qkv[i].split([HD, KD, KD], 1)
            self.attn.forward(q.view(T, -1, self.D), k.view(T, -1, self.D), v.view(T, -1, self.D),
                              self.cache, self.win_off, self.parent, layer=i, out=self.o)
            oq = ops.quantize_q8_k(self.o.view(T, HD))
            y = ops.gemv_q4_k_q8_f16out_batched(self.w_o[i], oq, H, HD, T)
        ops.add_rmsnorm_q8_k(self.x, self.norm[-1], 1e-6, y=y, x_out=self.x, xq=self.xq)
        ops.gemv_q4_k_q8_batched(self.w_head, self.xq, self.V, H, T, y=self.logits)
        self.verify.forward(self.logits, self.tokens, self.win_off, self.parent, self.temp, self.u,
                            self.us, None, *self.out)
        k, v = (self.qkv[:, :, a:a + KD].view(self.layers, T, self.KV, self.D)
                for a in (HD, HD + KD))
        self.cache.commit(k, v, self.win_off, self.out[0], self.out[1], length_out=self.length)

    def results(self):
        return [t.clone() for t in (self.x, self.o, self.logits, *self.out, self.length,
                                    self.cache.k, self.cache.v)]


def test_a_window_step_together():
    st = Step(3, [4, 1, 5], [20, 0, 77])
    st.run()
    r = st.results()
    # the attention and the verification of what the step itself computed
    i = st.layers - 1
    q = st.qkv[i].cpu().numpy()
    HD, KD, T = st.HEADS * st.D, st.KV * st.D, st.T
    par = st.parent.cpu().numpy()
    before = Step(3, [4, 1, 5], [20, 0, 77]).cache
    want, spread = ref.attention(
        q[:, :HD].reshape(T, -1, st.D), q[:, HD:HD + KD].reshape(T, -1, st.D),
        q[:, HD + KD:].reshape(T, -1, st.D), before.k[i].cpu().numpy(), before.v[i].cpu().numpy(),
        before.pages.cpu().numpy(), before.length.cpu().numpy(), st.off, par, st.D ** -0.5, 16,
        np.zeros((T, st.HEADS, st.D)))
    # scores: (D + 4) u32 of scale * sum |q k|
    top = float(np.abs(q[:, :HD]).max()) * float(max(np.abs(q[:, HD:]).max(), 5)) * st.D ** 0.5
    tol = U16 * np.abs(want) + (U16 + 100 * U32 + 68 * U32 * top) * spread + 1e-6
    assert (np.abs(r[1].float().cpu().numpy() - want) <= tol).all()
    want = ref.verify(r[2].cpu().numpy(), st.tokens.cpu().numpy(), st.off, par,
                      st.temp.cpu().numpy(), st.u.cpu().numpy(), st.us.cpu().numpy(), max_window=st.W)
    for g, w in zip(r[3:6], want[:3]):
        np.testing.assert_array_equal(g.cpu().numpy(), w)
    assert torch.equal(r[7], st.cache.length + r[4])


def test_a_window_step_in_a_graph():
    """Captured once, replayed with eager steps between the replays and new inputs."""
    eager = Step(4, [3, 2, 4], [33, 60, 5])
    st = Step(4, [3, 2, 4], [33, 60, 5])
    st.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st.run()
    for i in range(4):
        x = torch.randn_like(st.x0)
        st.x0.copy_(x)
        eager.x0.copy_(x)
        st.u.uniform_()
        eager.u.copy_(st.u)
        g.replay()
        eager.run()
        torch.cuda.synchronize()
        for a, b in zip(st.results(), eager.results()):  # (bits: a row may hold NaN)
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        for s in (st, eager):  # the next step's caches
            s.cache.length.copy_(torch.tensor([33 + i, 60 - i, 5 * i], dtype=torch.int32))


def test_same_call_twice_is_bit_equal():
    c = attn_case(51, [5, 7], [3000, 170], 2, 4, 128, 16, branch=3)
    op, cache = attn_op(c)
    first = run_attn(c, op, cache)
    for _ in range(3):
        assert torch.equal(first, run_attn(c, op, cache))
    c = verify_case(52, [6, 6, 3], 9001, branch=2, sampled=True)
    first = run_verify(c)
    for _ in range(3):
        assert all(np.array_equal(a, b) for a, b in zip(first, run_verify(c)))


def test_workspaces_are_checked():
    c = attn_case(61, [2], [4000], 1, 1, 64, 16, chain=True)
    op, cache = attn_op(c)
    assert op.workspace.numel() > 0
    with pytest.raises(ops.SagerError, match="workspace"):
        op.forward(dev(c["q"]), dev(c["k"]), dev(c["v"]), cache, dev(c["off"]),
                   workspace=op.workspace[:-16])
    with pytest.raises(ops.SagerError, match="aligned"):
        big = torch.zeros(op.workspace.numel() + 16, dtype=torch.uint8, device="cuda")
        op.forward(dev(c["q"]), dev(c["k"]), dev(c["v"]), cache, dev(c["off"]), workspace=big[4:])
    assert ctypes.sizeof(cache.desc) == 64
