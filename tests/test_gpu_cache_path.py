"""Rotary positions, the caches and the sliding attention together, as a model's layers use them: a
prompt's ragged chunks, then windows of drafted trees whose accepted line is committed, eagerly and
as a graph.

The caches' contents are compared exactly (what the rotary kernel wrote, quantised by the rule),
attention with the tolerance of its own tests, over what the caches hold."""
import numpy as np
import pytest
import torch

import cache_ref as cref
import test_gpu_window as w
import window_ref as ref
from sager_amd import ops

pytestmark = pytest.mark.gpu
dev = w.dev
LAYERS, PAGE, PER = 3, 16, 12


class Path:
    """Two sequences' caches, three layers of attention, tokens' projections at random."""

    def __init__(self, q8, n_kv, group, D, reach, sinks, max_window):
        self.q8, self.n_kv, self.H, self.D = q8, n_kv, n_kv * group, D
        self.reach, self.sinks = reach, sinks
        rng = np.random.default_rng(D)
        n = 2 * PER + 3
        self.pages = rng.permutation(n)[:2 * PER].reshape(2, PER).astype(np.int32)
        pages, length = dev(self.pages), dev(np.zeros(2, np.int32))
        if q8:
            self.cache = ops.KvCacheQ8.empty(LAYERS, n, n_kv, PAGE, D, pages, length)
        else:
            k, v = (torch.zeros((LAYERS, n, n_kv, PAGE, D), dtype=torch.float16, device="cuda")
                    for _ in range(2))
            self.cache = ops.KvCache(k, v, pages, length)
        # of chunks, and of trees (which have at most 64 nodes)
        self.chains, self.trees = (
            ops.SlidingAttention(self.H, n_kv, D, max_tokens=200, max_seqs=2, max_window=most,
                                 max_len=PAGE * PER, reach=reach, sinks=sinks)
            for most in (max_window, 5))
        self.max_window = max_window
        self.table = ops.rope_frequencies(D // 2, 10000.0)
        self.norms = [dev(rng.uniform(0.5, 1.5, D).astype(np.float32)) for _ in range(2)]
        # all tokens of the two caches, in the plain form's pool: K and V of a layer as values
        self.held = [[np.zeros((LAYERS, 0, n_kv, D)) for _ in range(2)] for _ in range(2)]

    def tokens(self, seed, n):
        rng = np.random.default_rng(seed)
        return dev(rng.normal(0, 1, (LAYERS, n, self.H + 2 * self.n_kv, self.D)).astype(np.float16))

    def layers(self, qkv, off, parent, out):
        """Positions and attention of every layer (the projections' rows change in place)."""
        H, K = self.H, self.n_kv
        attn = self.chains if parent is None else self.trees
        for l in range(LAYERS):
            q, k, v = qkv[l, :, :H], qkv[l, :, H:H + K], qkv[l, :, H + K:]
            ops.rope(q, k, self.table, win_off=off, parent=parent, length=self.cache.length,
                     q_norm=self.norms[0], k_norm=self.norms[1])
            attn.forward(q, k, v, self.cache, off, parent, layer=l, out=out[l])
        return qkv[:, :, H:H + K], qkv[:, :, H + K:]

    # ---- the plain form ----

    def check_rope(self, raw, done, off, parent, length):
        pos = cref.positions(off, parent, length, raw.shape[1])
        H, K = self.H, self.n_kv
        here = pos >= 0
        for l in range(LAYERS):
            for a, b, wt in ((0, H, 0), (H, H + K, 1)):
                x, y = raw[l, here, a:b], done[l, here, a:b].astype(np.float64)
                want, size = cref.rope(x, self.norms[wt].cpu().numpy(), 1e-6,
                                       self.table.cpu().numpy(), pos[here], False, 1.0)
                # half a step of the result; below it, fp32: the norm (some D + 8 roundings of
                # its sum, halved by the root, and four of its own) and the turn (eight)
                tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + (self.D / 2 + 16) * 2.0 ** -24 * size
                assert (np.abs(y - want) <= tol).all()
        assert (done[:, ~here] == raw[:, ~here]).all()
        assert (done[:, :, H + K:] == raw[:, :, H + K:]).all()

    def check_attention(self, done, off, parent, length, out):
        H, K = self.H, self.n_kv
        n = max(self.held[s][0].shape[1] for s in range(2))
        one = -(-max(n, 1) // PAGE)
        for l in range(LAYERS):
            kc, vc = (np.zeros((2 * one, K, PAGE, self.D)) for _ in range(2))
            pages = np.arange(2 * one, dtype=np.int32).reshape(2, one)
            for s in range(2):
                for c, pool in zip(self.held[s], (kc, vc)):
                    rows = np.zeros((one * PAGE, K, self.D))
                    rows[:c.shape[1]] = c[l]
                    pool[pages[s]] = rows.reshape(one, PAGE, K, self.D).transpose(0, 2, 1, 3)
            q, k, v = done[l, :, :H], done[l, :, H:H + K], done[l, :, H + K:]
            want, spread = cref.attention(q, k, v, kc, vc, pages, length, off, parent,
                                          self.D ** -0.5, PAGE, np.full(q.shape, 3.0), self.reach,
                                          self.sinks, self.max_window)
            c = dict(q=q, max_len=n, max_window=self.max_window, scale=self.D ** -0.5)
            assert (np.abs(out[l] - want) <= w.attn_tol(c, want, spread)).all()
            assert (out[l, off[-1]:] == 3.0).all()

    def hold(self, done, rows):
        """rows[s]: the rows of `done` that sequence s keeps."""
        H, K = self.H, self.n_kv
        for s in range(2):
            for i, x in enumerate((done[:, rows[s], H:H + K], done[:, rows[s], H + K:])):
                x = cref.values(*cref.quantise(x)) if self.q8 and x.size else x.astype(np.float64)
                self.held[s][i] = np.concatenate([self.held[s][i], x], 1)

    def check_cache(self):
        n = [self.held[s][0].shape[1] for s in range(2)]
        assert self.cache.length.tolist() == n
        off = ref.off_of(n)
        want = [np.concatenate([self.held[s][i] for s in range(2)], 1).astype(np.float16)
                for i in range(2)]
        if self.q8:
            got = self.cache.read(dev(np.zeros(2, np.int32)), dev(off), int(off[-1]))
        else:
            got = [torch.cat([t[:, self.cache.pages[s].long()].transpose(2, 3).flatten(1, 2)[:, :n[s]]
                              for s in range(2)], 1) for t in (self.cache.k, self.cache.v)]
        for a, b in zip(got, want):
            assert (a.cpu().numpy() == b).all()


def run(p, seed, sizes, parent, pad, keep):
    """One step: windows of `sizes`, then what keep(off) says is kept of them (None: all)."""
    off = ref.off_of(sizes)
    T = int(off[-1]) + pad
    length = p.cache.length.cpu().numpy()
    qkv = p.tokens(seed, T)
    raw = qkv.cpu().numpy()
    out = torch.full((LAYERS, T, p.H, p.D), 3.0, dtype=torch.float16, device="cuda")
    d_off, d_par = dev(off), None if parent is None else dev(parent)
    k, v = p.layers(qkv, d_off, d_par, out)
    if keep is None:
        rows = [np.arange(off[s], off[s + 1]) for s in range(2)]
        new = p.cache.append(k, v, d_off, max(sizes))
    else:
        path, n_path = keep
        rows = [off[s] + path[s, :n_path[s]] for s in range(2)]
        new = p.cache.commit(k, v, d_off, dev(path), dev(n_path))
    p.cache.length.copy_(new)
    done = qkv.cpu().numpy()
    p.check_rope(raw, done, off, parent, length)
    p.check_attention(done, off, parent, length, out.cpu().numpy().astype(np.float64))
    p.hold(done, rows)
    p.check_cache()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("n_kv,group,D,reach,sinks", [(2, 4, 64, 0, 0), (1, 8, 128, 40, 4),
                                                      (2, 2, 256, 70, 20)])
def test_a_conversation(q8, n_kv, group, D, reach, sinks):
    """A first chunk of one sequence, chunks of both, single tokens, trees with absent nodes."""
    p = Path(q8, n_kv, group, D, reach, sinks, max_window=70)
    run(p, 1, [33, 0], None, 0, None)
    run(p, 2, [70, 19], None, 2, None)
    run(p, 3, [1, 1], None, 0, None)
    tree = np.array([-1, 0, 0, 1, 2, -1, 0, 1, -2, 0, 0], np.int32)
    path, n_path = np.array([[0, 2, 4, 9, 9], [0, 1, 2, 9, 9]], np.int32), np.array([3, 2], np.int32)
    run(p, 4, [5, 4], tree, 2, (path, n_path))
    run(p, 5, [2, 3], None, 0, None)


@pytest.mark.parametrize("q8", [False, True])
def test_a_verify_step_as_a_graph(q8):
    """Positions, attention and commit of a window of every layer, the new lengths copied where the
    next step reads them: each replay goes on from the last and does what an eager step does."""
    sizes, rng = [5, 4], np.random.default_rng(5)
    off = ref.off_of(sizes)
    parent = np.array([-1, 0, 0, 1, 2, -1, 0, 1, 2], np.int32)
    pair = [Path(q8, 2, 4, 128, 50, 4, 64) for _ in range(2)]
    first = [pair[0].tokens(1, 90).cpu().numpy()] * 2
    for p, x in zip(pair, first):
        o = dev(np.array([0, 50, 90], np.int32))
        H, K = p.H, p.n_kv
        x = dev(x)
        p.cache.length.copy_(p.cache.append(x[:, :, H:H + K], x[:, :, H + K:], o, 50))
    d_off, d_par = dev(off), dev(parent)
    bufs = [dict(raw=p.tokens(2, 9), out=torch.zeros(LAYERS, 9, p.H, p.D, dtype=torch.float16, device="cuda"),
                 path=torch.zeros(2, 5, dtype=torch.int32, device="cuda"),
                 n=torch.zeros(2, dtype=torch.int32, device="cuda"),
                 new=torch.zeros(2, dtype=torch.int32, device="cuda")) for p in pair]
    for b in bufs:
        b["qkv"] = torch.zeros_like(b["raw"])

    def step(p, b):
        b["qkv"].copy_(b["raw"])
        k, v = p.layers(b["qkv"], d_off, d_par, b["out"])
        p.cache.commit(k, v, d_off, b["path"], b["n"], length_out=b["new"])
        p.cache.length.copy_(b["new"])

    step(pair[0], bufs[0])  # (nothing accepted: the caches stay alike)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(pair[0], bufs[0])
    for turn in range(4):
        raw = pair[0].tokens(10 + turn, 9)
        path = np.array([[0, 2, 4, 0, 0], [0, 1, 2, 3, 0]], np.int32)
        n = rng.integers(0, 4, 2).astype(np.int32)
        for b in bufs:
            b["raw"].copy_(raw)
            b["path"].copy_(dev(path))
            b["n"].copy_(dev(n))
        g.replay()
        step(pair[1], bufs[1])
        torch.cuda.synchronize()
        for name in ("qkv", "out", "new"):
            assert torch.equal(bufs[0][name], bufs[1][name]), (turn, name)
        for name, t in pair[0].cache._tensors.items():
            assert torch.equal(t, pair[1].cache._tensors[name]), (turn, name)


# (256 heads behind what may be a long cache get blocks of 256 rows)
@pytest.mark.parametrize("heads,max_len", [(1, 2), (16, 2), (128, 2), (256, 10 ** 6)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [8, 0, -9, -14])
def test_quantised_keys_are_not_rounded(power, D, heads, max_len):
    """Keys whose values, 128 1/16 and 128 3/16 times a power of two, lie half a step of 16 bits from
    the next, one below and one above: their scores are 256 and 256 1/4, and 256 1/2 if keys were
    rounded, which moves the weights by 6 %.  A score's sum of 256 is off by 2 D roundings of 2^-24 at
    the most, that is, the weights by D 2^-15."""
    q = np.ones((1, heads, D), np.float16)
    kc = np.zeros((1, 2, 1, 16, D), np.int8)
    vc = np.random.default_rng(0).integers(-127, 128, kc.shape).astype(np.int8)
    ks, vs = (np.ones((1, 2, 1, 16, D // 32), np.float16) for _ in range(2))
    for j, (code, m, half) in enumerate(((96, 342, slice(0, D // 2)), (112, 148, slice(D // 2, D)))):
        ks[0, 1, 0, j] = (1 + m / 1024) * 2.0 ** power
        assert float(ks[0, 1, 0, j, 0]) == (1 + m / 1024) * 2.0 ** power
        kc[0, 1, 0, j, half] = code
    k, v = np.zeros((1, 1, D), np.float16), np.ones((1, 1, D), np.float16)
    pages, length = np.array([[1]], np.int32), np.array([2], np.int32)
    cache = ops.KvCacheQ8(*(dev(x) for x in (kc, vc, ks, vs, pages, length)))
    op = ops.SlidingAttention(heads, 1, D, max_tokens=1, max_len=max_len)
    by = 256 / (2.0 ** power * 128.0625 * D / 2)
    got = op.forward(dev(q), dev(k), dev(v), cache, dev(np.array([0, 1], np.int32)),
                     scale=by).cpu().numpy().astype(np.float64)
    args = cref.values(vc, vs)[0], pages, length, np.array([0, 1]), None, by, 16, np.zeros(q.shape)
    exact = cref.values(kc, ks)[0]
    want, spread = cref.attention(q, k, v, exact, *args)
    tol = 2.0 ** -11 * np.abs(want) + (2.0 ** -11 + D * 2.0 ** -15) * spread
    assert (np.abs(got - want) <= tol).all()
    rounded, _ = cref.attention(q, k, v, exact.astype(np.float16), *args)
    assert (np.abs(rounded - want) > tol).any()  # (what the test would find)


def test_a_cache_keeps_its_tensors():
    pages, length = dev(np.zeros((2, 3), np.int32)), dev(np.zeros(2, np.int32))
    c = ops.KvCacheQ8.empty(2, 4, 1, 16, 64, pages, length)
    assert c.k.shape == c.v.shape == (2, 4, 1, 16, 64) and c.k.dtype == torch.int8
    assert c.k_scale.shape == c.v_scale.shape == (2, 4, 1, 16, 2) and c.pages is pages
    for name in ("k", "v", "k_scale", "v_scale", "pages", "length"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name).clone())
    for bad in (dict(k=c.v.half()), dict(k_scale=c.v_scale.float()), dict(v_scale=c.k_scale[..., :1]),
                dict(pages=pages.long()), dict(length=length[:1]), dict(pages=pages.cpu()),
                dict(v=c.k[:, :2])):
        with pytest.raises(ops.SagerError):
            ops.KvCacheQ8(**{**c._tensors, **bad})
