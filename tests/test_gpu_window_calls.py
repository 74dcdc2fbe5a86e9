"""Calls of the verify window's operators that lie past the sizes of test_gpu_window.py: many
sequences, aliases, subnormal temperatures, workspaces and graphs shared by calls, refusals of the
Python layer."""
import numpy as np
import pytest
import torch

import test_gpu_window as w
import window_ref as ref
from sager_amd import ops

pytestmark = pytest.mark.gpu
dev = w.dev


# ---- residual, norm, Q8_K -----------------------------------------------------

@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
@pytest.mark.parametrize("n", [256, 2048, 8448])
def test_add_rmsnorm_aliases(dt, n):
    """x_out over x or y, xn over the other; xn over x where nothing is added."""
    g = torch.Generator(device="cuda").manual_seed(n)
    x, y = (torch.randn(37, n, generator=g, device="cuda").to(dt) for _ in range(2))
    wt = torch.rand(n, generator=g, device="cuda") + 0.5
    r, xn, xq = ops.add_rmsnorm_q8_k(x, wt, 1e-6, y=y)
    for swap in (False, True):
        a, b = x.clone(), y.clone()
        q = torch.empty_like(xq)
        ops.add_rmsnorm_q8_k(a, wt, 1e-6, y=b, x_out=b if swap else a, xn=a if swap else b, xq=q)
        assert torch.equal(b if swap else a, r) and torch.equal(a if swap else b, xn)
        assert torch.equal(q, xq)
    a = r.clone()
    _, got, _ = ops.add_rmsnorm_q8_k(a, wt, 1e-6, xn=a)
    assert torch.equal(got, xn) and got is a


def test_add_rmsnorm_many_rows():
    """More rows than a launch's 65,536 in other dimensions would be."""
    x = torch.randn(70001, 256, device="cuda").half()
    wt = torch.ones(256, device="cuda")
    _, xn, xq = ops.add_rmsnorm_q8_k(x, wt, 1e-6)
    _, tail, tail_q = ops.add_rmsnorm_q8_k(x[-3:].clone(), wt, 1e-6)
    assert torch.equal(xn[-3:], tail) and torch.equal(xq[-3:], tail_q)


# ---- attention ------------------------------------------------------------------

@pytest.mark.parametrize("n_seq,longest", [(65, 300), (65, 3000), (200, 90), (600, 100),
                                           (600, 900)])
def test_attention_of_many_sequences(n_seq, longest):
    """More sequences than a wave has lanes, cut into parts and not, some without a window, some
    without a cache; the window of the longest in the middle of the batch."""
    rng = np.random.default_rng(n_seq + longest)
    sizes = [int(x) for x in rng.integers(0, 3, n_seq)]
    lengths = [int(x) for x in rng.integers(0, 70, n_seq)]
    sizes[n_seq // 2], lengths[n_seq // 2] = 2, longest
    sizes[-1], lengths[-1] = 1, longest // 2
    w.check_attn(w.attn_case(7, sizes, lengths, 2, 1, 64, 16, chain=True, pad=2))


@pytest.mark.parametrize("n_seq,n_kv,D,longest", [(66, 8, 256, 1500), (60, 18, 128, 2100),
                                                  (66, 8, 256, 5)])
def test_attention_of_more_than_two_rounds(n_seq, n_kv, D, longest):
    """As many heads of sequences as twice the workgroups the card holds: only the longest are cut,
    and some sequences have neither a window nor a cache."""
    rng = np.random.default_rng(D + longest)
    sizes = [int(x) for x in rng.integers(0, 3, n_seq)]
    lengths = [int(x) for x in rng.integers(0, min(longest, 70), n_seq)]
    for i in (0, n_seq // 2, n_seq - 1):
        sizes[i], lengths[i] = 1 + i % 2, longest - i
        lengths[i] = max(lengths[i], 0)
    w.check_attn(w.attn_case(19, sizes, lengths, n_kv, 1, D, 16, chain=True, pad=1))


def test_attention_with_a_workspace_for_more_sequences():
    """The workspace of a large batch, which is not cut, serves small ones, which are."""
    for sizes, lengths in (([3, 1, 2], [400, 90, 333]), ([64], [500]), ([1] * 9, [450] * 9)):
        c = w.attn_case(13, sizes, lengths, 2, 4, 128, 16, branch=2)
        T, heads, D = c["q"].shape
        cache = ops.KvCache(dev(c["kc"]), dev(c["vc"]), dev(c["pages"]), dev(c["length"]))
        op = ops.TreeAttention(heads, 2, D, max_tokens=9000, max_seqs=700, max_window=64,
                               max_len=500)
        got = w.run_attn(c, op, cache).cpu().numpy().astype(np.float64)
        want, spread = ref.attention(c["q"], c["k"], c["v"], c["kc"][0], c["vc"][0], c["pages"],
                                     c["length"], c["off"], c["parent"], c["scale"], 16,
                                     np.zeros(c["q"].shape))
        assert (np.abs(got - want) <= w.attn_tol(c, want, spread)).all()


def test_attention_without_a_score():
    """A node all of whose scores are -infinity gets 0, the others are what they were."""
    for group in (1, 40):
        c = w.attn_case(17, [3], [0], 1, group, 64, 16, chain=True)
        base = w.run_attn(c).cpu().numpy()
        c["q"][0, :, 0], c["k"][0, 0, 0] = 1, -np.inf
        c["q"][1:, :, 0] = 0
        d = {k: np.copy(v) if isinstance(v, np.ndarray) else v for k, v in c.items()}
        d["parent"] = np.array([-1, -1, 1], np.int32)  # nodes 1 and 2 hang on nothing
        got = w.run_attn(d).cpu().numpy()
        assert (got == 0).all() and np.isfinite(base).all()


def test_attention_on_two_streams_and_in_two_graphs():
    """Two calls under way at once, each with its workspace; two graphs that share one, replayed in
    turn on one stream, with eager calls in between."""
    cs = [w.attn_case(s, [5, 3], [2500, 900], 2, 4, 128, 16, branch=2) for s in (71, 72)]
    ops_ = [w.attn_op(c) for c in cs]
    want = [w.run_attn(c, *o) for c, o in zip(cs, ops_)]
    args = [[dev(c[n]) for n in ("q", "k", "v")] for c in cs]
    rest = [(dev(c["off"]), dev(c["parent"])) for c in cs]
    outs = [torch.zeros_like(o) for o in want]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                ops_[i][0].forward(*args[i], ops_[i][1], *rest[i], scale=cs[i]["scale"],
                                   out=outs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    op = ops_[0][0]
    graphs = []
    for i in range(2):
        outs[i].zero_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            op.forward(*args[i], ops_[i][1], *rest[i], scale=cs[i]["scale"], out=outs[i])
        graphs.append(g)
    for _ in range(3):
        for i, g in enumerate(graphs):
            outs[i].zero_()
            g.replay()
            assert torch.equal(w.run_attn(cs[1 - i], op, ops_[1 - i][1]), want[1 - i])
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i])


# ---- verification -----------------------------------------------------------------

@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("t", [2.0 ** -126, 1e-40, 1.5e-45, 1e-30, 1e30, np.inf])
def test_verify_extreme_temperatures(sampled, t):
    """Down to the least subnormal number, where all the mass is on the largest logits; up to
    infinity, where it is spread evenly."""
    c = w.verify_case(81, [4, 6, 1], 301, branch=2, sampled=sampled, temps=(t,))
    c["logits"][2, [5, 70, 71]] = 50.0   # equals share
    c["logits"][5] = np.round(c["logits"][5])
    w.check_verify(c)


@pytest.mark.parametrize("sampled", [False, True])
def test_verify_more_chunks_than_threads(sampled):
    """A vocabulary of over four million; the last token among its first, middle and last."""
    c = w.verify_case(82, [2], 4096 * 1024 + 4097, chain=True, sampled=sampled, peak=0.0)
    for u in (0.0, 0.5, 1 - 2.0 ** -24):
        c["u_smp"][:] = u
        w.check_verify(c)


@pytest.mark.parametrize("vocab,window,n_seq", [(8200, 12, 57), (4097, 16, 64)])
def test_verify_of_several_rounds(vocab, window, n_seq):
    """So many blocks of logits that a workgroup takes two of them, an odd number a row and an even
    one."""
    assert -(-vocab // 4096) * window * n_seq >= 2048
    c = w.verify_case(85, [window - i % 5 for i in range(n_seq)], vocab, branch=3, absent=True,
                      sampled=True, peak=3.0)
    w.check_verify(c, 3)


def test_verify_in_two_graphs_with_one_workspace():
    cs = [w.verify_case(s, [6, 4], 9001, branch=2, sampled=True) for s in (83, 84)]
    op = ops.TreeVerify(9001, max_tokens=10, max_seqs=2, max_window=6, max_children=2)
    want = [w.run_verify(c, op=op) for c in cs]
    names = ("logits", "tokens", "off", "parent", "temp", "u_acc", "u_smp", "draft")
    args = [[dev(c[n]) for n in names] for c in cs]
    outs, graphs = [], []
    for i in range(2):
        kw = dict(path=torch.zeros((2, 6), dtype=torch.int32, device="cuda"),
                  prob=torch.full((10,), 5.0, device="cuda"))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(op.forward(*args[i], **kw))
        graphs.append(g)
    for _ in range(3):
        for i, g in enumerate(graphs):
            for t in outs[i][:3]:
                t.fill_(77)
            g.replay()
            w.run_verify(cs[1 - i], op=op)
            torch.cuda.synchronize()
            for a, b in zip(outs[i], want[i]):
                np.testing.assert_array_equal(a.cpu().numpy(), b)


# ---- refusals of the Python layer ---------------------------------------------------

def refused(fn, *args, **kw):
    with pytest.raises(ops.SagerError):
        fn(*args, **kw)


def test_norm_arguments():
    x, wt = torch.zeros(4, 512, device="cuda").half(), torch.ones(512, device="cuda")
    f = ops.add_rmsnorm_q8_k
    refused(f, x.cpu(), wt, 1e-6)
    refused(f, x, wt.cpu(), 1e-6)
    refused(f, x, wt.half(), 1e-6)
    refused(f, x, wt[:256], 1e-6)
    refused(f, x.double(), wt, 1e-6)
    refused(f, x[:, :300], torch.ones(300, device="cuda"), 1e-6)
    refused(f, x[:, ::2], wt[::2].contiguous(), 1e-6)
    refused(f, x, wt, 1e-6, y=x.float())
    refused(f, x, wt, 1e-6, y=x[:2])
    refused(f, x, wt, 1e-6, x_out=x)
    refused(f, x, wt, 1e-6, xn=x.float())
    refused(f, x, wt, 1e-6, xq=ops.q8k_empty(3, 512))
    refused(f, x, wt, 1e-6, xq=ops.q8k_empty(4, 512, "cpu"))
    refused(f, x[:0], wt, 1e-6)
    refused(f, x.new_zeros(()), wt, 1e-6)


def test_attention_and_commit_arguments():
    c = w.attn_case(91, [3], [40], 2, 2, 64, 16, chain=True)
    op, cache = w.attn_op(c, max_len=5000)
    q, k, v, off = (dev(c[n]) for n in ("q", "k", "v", "off"))
    par = torch.zeros(3, dtype=torch.int32, device="cuda")
    op.forward(q, k, v, cache, off, par)
    refused(op.forward, q.cpu(), k, v, cache, off)
    refused(op.forward, q, k.cpu(), v, cache, off)
    refused(op.forward, q.float(), k, v, cache, off)
    refused(op.forward, q[:, :2], k, v, cache, off)
    refused(op.forward, q, k[:2], v, cache, off)
    refused(op.forward, q, k.transpose(0, 1).contiguous().transpose(0, 1), v, cache, off)
    refused(op.forward, q, k, v[:1].expand(3, 2, 64), cache, off)
    refused(op.forward, q, k, v, cache, off.long())
    refused(op.forward, q, k, v, cache, off[:1])
    refused(op.forward, q, k, v, cache, off, par[:2])
    refused(op.forward, q, k, v, cache, off, par, layer=1)
    refused(op.forward, q, k, v, cache, off, par, out=torch.empty_like(q).float())
    refused(op.forward, q, k, v, cache, off, par, workspace=op.workspace.cpu())
    refused(op.forward, q, k, v, cache, off, par, workspace=op.workspace[:1].expand(1 << 24))
    refused(op.forward, *(torch.cat([t, t]) for t in (q, k, v)), cache, off)
    refused(op.forward, q, k, v, cache, torch.zeros(3, dtype=torch.int32, device="cuda"))
    other = ops.KvCache(*(torch.zeros(1, 4, 1, 16, 64, device="cuda").half() for _ in range(2)),
                        cache.pages, cache.length)
    refused(op.forward, q, k, v, other, off)
    refused(ops.TreeAttention, 3, 2, 64, 8)
    refused(ops.KvCache, cache.k, cache.v[:, :1], cache.pages, cache.length)
    refused(ops.KvCache, cache.k, cache.v, cache.pages.long(), cache.length)
    refused(ops.KvCache, cache.k, cache.v, cache.pages, cache.length.cpu())
    path = torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    n = torch.ones(1, dtype=torch.int32, device="cuda")
    cache.commit(k[None], v[None], off, path, n)
    refused(cache.commit, k, v, off, path, n)
    refused(cache.commit, k[None], v[None, :2], off, path, n)
    refused(cache.commit, k[None].float(), v[None], off, path, n)
    refused(cache.commit, k[None], v[None], off, path[0], n)
    refused(cache.commit, k[None], v[None], off, path, n.long())
    refused(cache.commit, k[None], v[None], off, path, n, length_out=cache.length)
    refused(cache.commit, k[None], v[None], off, path, n, length_out=n.cpu())


def test_verify_arguments():
    c = w.verify_case(92, [3, 2], 300, sampled=True)
    names = ("logits", "tokens", "off", "parent", "temp", "u_acc", "u_smp", "draft")
    good = [dev(c[n]) for n in names]
    op = ops.TreeVerify(300, max_tokens=5, max_seqs=2, max_window=3, max_children=1)
    op.forward(*good)
    for i in range(len(names)):
        for bad in (good[i].cpu(), good[i].double(), good[i][:-1]):
            refused(op.forward, *good[:i], bad, *good[i + 1:])
    refused(op.forward, *good, prob=torch.zeros(5, device="cuda").double())
    refused(op.forward, *good, path=torch.zeros(2, 4, dtype=torch.int32, device="cuda"))
    refused(op.forward, *good, workspace=op.workspace[:-16])
    refused(op.forward, *good, workspace=op.workspace.cpu())
    refused(ops.TreeVerify(300, 5, 2, 3).forward, *good)            # no max_children
    refused(ops.TreeVerify(300, 5, 1, 3, 1).forward, *good)         # two sequences
    refused(ops.TreeVerify(299, 5, 2, 3, 1).forward, *good)
