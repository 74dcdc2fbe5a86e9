"""What a key brings to a row of the sliding attention, closely: single keys' weights, quantised values
that would be seen if they were rounded, and sums of the weights that the products are made with."""
import numpy as np
import pytest
import torch

import cache_ref as cref
import test_gpu_sliding as sl
import test_gpu_sliding_rows as rows
import test_gpu_window as w
from sager_amd import ops

pytestmark = pytest.mark.gpu
dev = w.dev
MARK = 254.0  # 127 * 2


def marked(c, seed):
    """V is 0 but for MARK in one column of each of the keys that are looked at: a sequence has as many
    as V has columns, those at borders among them.  So an output is a single key's weight."""
    rng = np.random.default_rng(seed)
    D, page, reach = c["q"].shape[2], c["page"], c["reach"] or 10 ** 9
    code, v = np.zeros(c["vc"].shape, np.int8), np.zeros_like(c["v"])
    for s, n in enumerate(c["length"]):
        a, b = int(c["off"][s]), int(c["off"][s + 1])
        size = b - a
        if size == 0:
            continue
        near = [0, 1, n - 1, n - 2, n - 16, n - 17, page - 1, page, c["sinks"] - 1, c["sinks"], 63, 64,
                n - reach, n - reach + 1, n - reach + size, n // 64 * 64, n // 64 * 64 - 1, n,
                n + 1, n + size - 1, n + size // 2, n + 63, n + 64]
        keys = list(dict.fromkeys(int(j) for j in near if 0 <= j < n + size))[:D]
        keys += rng.integers(0, n + size, D - len(keys)).tolist()
        for col, j in zip(rng.permutation(D), keys):
            if j < n:
                code[0, c["pages"][s, j // page], :, j % page, col] = 127
            else:
                v[a + j - n, :, col] = MARK
    c["v"], c["vc"] = v, (code != 0) * np.float16(MARK)
    if c["q8"]:
        c["codes"][1] = code, np.full((*code.shape[:-1], D // 32), 2, np.float16)
        assert (cref.values(*c["codes"][1]) == c["vc"]).all()
    return c


def look(c, max_len=None):
    """The tolerance: the weight's, the sum's and the output's rounding, 2^-11 each; a score's sum of 2 D
    products in fp32 and the steps that scale it; weights below 2^-22 of the largest are off by 2^-33 of it,
    and the output's last bit is 2^-24.  With the cached keys 0.4 % larger, it would not do."""
    op, cache = sl.make(c, max_len)
    T, heads, D = c["q"].shape
    got = w.run_attn(c, op, cache, out=torch.zeros((T, heads, D), dtype=torch.float16, device="cuda"))
    got = got.cpu().numpy().astype(np.float64)
    want, _ = sl.plain(c, np.zeros(c["q"].shape))
    q, k, kc = (np.abs(c[n].astype(np.float64)) for n in ("q", "k", "kc"))
    norm = [np.sqrt((x * x).sum(-1)).max() for x in (q, k, kc)]
    top = abs(c["scale"]) * norm[0] * max(norm[1:])  # no less than any sum of |q k|
    n = c["length"].max() + c["max_window"]
    rel = 3 * 2.0 ** -11 + 2 * (2 * D * 2.0 ** -24 + 4 * 2.0 ** -23) * top + (n + 100) * 2.0 ** -24
    tol = rel * want + 2.0 ** -24
    assert ((got == 0) | (want != 0)).all()  # keys that are not seen bring nothing
    bad = np.abs(got - want) - tol
    assert (bad <= 0).all(), (bad.max(), np.argwhere(bad > 0)[:5])
    if c["length"].max() > 100:
        more, _ = sl.plain({**c, "kc": c["kc"].astype(np.float64) * 1.004}, np.zeros(c["q"].shape))
        assert (np.abs(more - want) > tol).any()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("reach,sinks", [(0, 0), (700, 4), (70, 130)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_weights(D, reach, sinks, q8):
    """Parts, trees with absent nodes, a chunk."""
    kw = dict(reach=reach, sinks=sinks, q8=q8)
    look(marked(sl.case(D, [3, 1, 4], [4000, 65, 1100], 2, 4, D, 64, branch=2, **kw), 1))
    look(marked(sl.case(D + 1, [13, 7, 1], [300, 64, 0], 1, 3, D, 16, branch=3, absent=True, **kw), 2))
    look(marked(sl.case(D + 2, [200, 65], [129, 77], 2, 1, D, 32, chain=True, **kw), 3))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("reach,sinks", [(0, 0), (100, 70)])
@pytest.mark.parametrize("D,n_kv,group", rows.SHAPES)
def test_weights_in_blocks_of_256_rows(D, n_kv, group, reach, sinks, q8):
    kw = dict(reach=reach, sinks=sinks, q8=q8, chain=True)
    c = sl.case(D, [200, 65] + [0] * 600, [300, 77] + [0] * 600, n_kv, group, D, 16, **kw)
    assert rows.wide(c)[:2] == (True, False)
    look(marked(c, 4))
    if reach == 0:
        c = sl.case(D + 1, [130], [900], n_kv, group, D, 32, **kw)
        assert rows.wide(c, 10 ** 6)[:2] == (True, True)
        look(marked(c, 5), 10 ** 6)


# blocks of 16 and of 32 rows, whole and in parts, of 256 (behind what may be a long cache)
FORMS = [(1, 2), (16, 2), (128, 2), (16, 10 ** 6), (256, 10 ** 6)]


def quantised(heads, D, max_len, kc, ks, vc, vs, n, q, k, v, scale):
    """heads rows of one token over n cached ones."""
    pages = np.arange(1, kc.shape[1], dtype=np.int32)[None]
    cache = ops.KvCacheQ8(*(dev(x) for x in (kc, vc, ks, vs, pages, np.array([n], np.int32))))
    op = ops.SlidingAttention(heads, 1, D, max_tokens=1, max_len=max_len)
    got = op.forward(dev(q), dev(k), dev(v), cache, dev(np.array([0, 1], np.int32)), scale=scale)
    return got.cpu().numpy().astype(np.float64), (pages, np.array([n], np.int32), np.array([0, 1]), None,
                                                  scale, 16, np.zeros(q.shape))


@pytest.mark.parametrize("heads,max_len", FORMS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [8, 0, -9, -14])
def test_quantised_values_are_not_rounded(power, D, heads, max_len):
    """Two cached keys of one score, whose values 128 1/16 and -128 3/16, times a power of two, lie half a
    step of 16 bits from the next: half their sum is -1/16, and -1/8 of rounded values.  The window's own
    key has a weight of 2^-128 or less.  Equal weights have equal roundings, so what is left is the
    output's and sums of fp32."""
    q, k = np.ones((1, heads, D), np.float16), np.full((1, 1, D), -4, np.float16)
    v = np.full((1, 1, D), 7, np.float16)
    kc, vc = (np.zeros((1, 2, 1, 16, D), np.int8) for _ in range(2))
    ks, vs = (np.ones((1, 2, 1, 16, D // 32), np.float16) for _ in range(2))
    sign = 1 - 2 * (np.arange(D) % 2)
    even = np.arange(D) // 32 % 2 == 0
    for j in range(2):  # (the larger one in the other groups)
        first = even == (j == 0)
        vc[0, 1, 0, j] = np.where(first, 96, 112) * sign * (1 - 2 * j)
        vs[0, 1, 0, j] = (np.where(first, 1 + 342 / 1024, 1 + 148 / 1024) * 2.0 ** power)[::32]
    got, args = quantised(heads, D, max_len, kc, ks, vc, vs, 2, q, k, v, 1.0)
    exact = cref.values(vc, vs)[0]
    assert set(np.abs(exact[1, 0, :2]).ravel()) == {128.0625 * 2.0 ** power, 128.1875 * 2.0 ** power}
    want, spread = cref.attention(q, k, v, cref.values(kc, ks)[0], exact, *args)
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -20 * spread
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
    rounded, _ = cref.attention(q, k, v, cref.values(kc, ks)[0], exact.astype(np.float16), *args)
    assert (np.abs(rounded - want) > tol).all()  # (what the test would find)


def near_a_tie(below):
    """code and scale, 1 + a / 1024, of a product 1/64 of a 16-bit step below or above a tie."""
    for code in range(127, 100, -1):
        for a in range(1023, 0, -1):
            if code * a % 128 == (62 if below else 66) and 128 <= code * (1 + a / 1024) < 256:
                return code, 1 + a / 1024


@pytest.mark.parametrize("heads,max_len", FORMS)
@pytest.mark.parametrize("n", [40, 100])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_weights_sum_to_one(D, n, heads, max_len):
    """All cached keys have one value, 1/64 of a step (2^-17 of it or more) beside where its rounding turns:
    the outputs are that value rounded if the sum is of the weights that the product is made with, since
    sums of fp32 are off by 100 2^-24 at the most.  With a sum of weights that are not rounded some heads
    are not so."""
    rng = np.random.default_rng(D + n + heads)
    pages = (n + 15) // 16
    q, k = rng.normal(0, 1, (1, heads, D)).astype(np.float16), np.zeros((1, 1, D), np.float16)
    q[..., 0], k[..., 0] = 8, -2000
    kc = rng.integers(-127, 128, (1, pages + 1, 1, 16, D)).astype(np.int8)
    kc[..., 0] = 0
    ks, vs = (np.full((*kc.shape[:-1], D // 32), 1 / 64, np.float16) for _ in range(2))
    vc = np.zeros_like(kc)
    for g in range(D // 32):
        code, scale = near_a_tie(g % 2 == 0)
        vc[..., 32 * g:32 * g + 32], vs[..., g] = code, scale
        assert float(vs[0, 0, 0, 0, g]) == scale
    v = np.full((1, 1, D), 100, np.float16)
    scale = D ** -0.5 * 2
    got, _ = quantised(heads, D, max_len, kc, ks, vc, vs, n, q, k, v, scale)
    value = cref.values(vc, vs)[0, 0, 0, 0]
    assert (np.abs(value / 2.0 ** -3 % 1 - 0.5) == 1 / 64).all()  # (steps of 1/8)
    want = value.astype(np.float16).astype(np.float64)
    assert (got == want).all()
    # the weights over a reference 8 below the largest, rounded, and their sum without that
    keys = cref.values(kc, ks)[0, 1:, 0].reshape(-1, D)[:n]
    s = q[0].astype(np.float64) @ keys.T * scale * np.log2(np.e)
    p = 2.0 ** (s - s.max(1, keepdims=True) + 8)
    off = (p.astype(np.float16).astype(np.float64).sum(1) / p.sum(1))[:, None] * value
    if heads > 1:
        assert (off.astype(np.float16) != want).any()
