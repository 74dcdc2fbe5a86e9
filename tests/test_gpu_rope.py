"""Heads' norms and rotary positions against their plain form in 64 bits.

Tolerances.  The result is rounded once to its type (half a step).  Before that, in fp32 (2^-24 a
rounding): an angle within half a turn as a float (half turns up to 1: 2^-25, times pi), sine and
cosine (2 units in the last place), mscale, two products and a sum, together less than 2^-21 of
(|a| + |b|) mscale; a norm's sum of 512 squares, its root, quotient and product less than 2^-20."""
import numpy as np
import pytest
import torch

import cache_ref as cref
import window_ref as ref
from sager_amd import ops

pytestmark = pytest.mark.gpu


def dev(x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()


def check(got, want, size, dtype):
    got = got.cpu().numpy().astype(np.float64)
    step = 2.0 ** -11 if dtype == np.float16 else 2.0 ** -24
    tiny = 2.0 ** -25 if dtype == np.float16 else 0
    bad = np.abs(got - want) > step * np.abs(want) + size * (2.0 ** -21 + 2.0 ** -20) + tiny
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


def case(rng, T, H, K, D, dtype, gap=3):
    """q and k as slices of one buffer, with rows that are not theirs around them."""
    buf = (rng.normal(0, 1.5, (T, (H + K) * D + gap))).astype(dtype)
    t = torch.from_numpy(buf).cuda()
    q, k = t[:, 1:1 + H * D].unflatten(1, (H, D)), t[:, 1 + H * D:1 + (H + K) * D].unflatten(1, (K, D))
    return buf, t, q, k


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("H,K,D,rot", [(16, 2, 256, 64), (32, 8, 128, 128), (3, 1, 80, 80),
                                       (5, 5, 96, 50), (1, 1, 8, 2), (7, 3, 64, 22), (2, 1, 512, 512),
                                       (40, 8, 24, 12)])
def test_given_positions(dtype, H, K, D, rot):
    rng = np.random.default_rng(H * D + rot)
    pos = np.array([0, 1, 7, 4099, 131071, 524287, 2 ** 31 - 1, -5, 65], np.int32)
    T = len(pos)
    wq, wk = (rng.normal(1, 0.2, D).astype(np.float32) for _ in range(2))
    table = ops.rope_frequencies(rot, 1e6)
    for nb in (False, True):
        for w in ((wq, wk), (None, wk), (None, None)):
            buf, t, q, k = case(rng, T, H, K, D, dtype)
            x = [a.cpu().numpy() for a in (q, k)]
            qo, ko = ops.rope(q, k, table, positions=dev(pos), interleaved=nb, mscale=1.25,
                              q_norm=dev(w[0]), k_norm=dev(w[1]), eps=1e-5)
            assert qo is q and ko is k
            for got, a, n in ((qo, x[0], w[0]), (ko, x[1], w[1])):
                want, size = cref.rope(a, n, 1e-5, cref.turns(rot, 1e6), pos, nb, 1.25)
                check(got, want, size, dtype)
            edge = t.cpu().numpy()
            assert (edge[:, 0] == buf[:, 0]).all() and (edge[:, -2:] == buf[:, -2:]).all()
            # into other buffers, the same bits; q alone
            out = torch.zeros(T, H, D, dtype=t.dtype, device="cuda")
            src = torch.from_numpy(x[0]).cuda()
            got, none = ops.rope(src, None, table, positions=dev(pos), interleaved=nb, mscale=1.25,
                                 q_norm=dev(w[0]), eps=1e-5, q_out=out)
            assert none is None and torch.equal(got, qo) and (src.cpu().numpy() == x[0]).all()


@pytest.mark.parametrize("sizes,lengths,branch,absent", [
    ([4], [4099], 1, False), ([1, 0, 7, 64, 13], [0, 3, 524287, 77, 100], 3, True),
    ([2] * 130, list(range(130)), 1, False), ([5, 0, 0, 9], [1, 2, 3, 4], 2, True)])
def test_windows(sizes, lengths, branch, absent):
    rng = np.random.default_rng(len(sizes))
    off, pad, H, K, D, rot = ref.off_of(sizes), 3, 4, 2, 64, 32
    T = int(off[-1]) + pad
    par = np.concatenate([ref.tree(rng, n, branch, absent) for n in sizes if n] + [[-1] * pad])
    par, length = par.astype(np.int32), np.array(lengths, np.int32)
    table = ops.rope_frequencies(rot, 1e4, "yarn", factor=4, trained=4096)
    tab = cref.turns(rot, 1e4, "yarn", 4, 4096)
    for p in (par, None):
        buf, _, q, k = case(rng, T, H, K, D, np.float16)
        x = [a.cpu().numpy() for a in (q, k)]
        pos = cref.positions(off, p, length, T)
        ops.rope(q, k, table, win_off=dev(off), parent=dev(p), length=dev(length))
        for got, a in ((q, x[0]), (k, x[1])):
            want, size = cref.rope(a, None, 0, tab, pos, False, 1.0)
            at = pos >= 0
            check(got[torch.from_numpy(at)], want[at], size[at], np.float16)
            assert (got.cpu().numpy()[~at] == a[~at]).all()


def test_a_long_chunk_and_many_sequences():
    """Chains past 64 rows, more sequences than 64 * 64."""
    rng = np.random.default_rng(5)
    for sizes in ([1000, 3, 70], [1] * 4200 + [2, 0, 5]):
        off, n = ref.off_of(sizes), len(sizes)
        length = rng.integers(0, 100000, n).astype(np.int32)
        x = rng.normal(0, 1, (int(off[-1]), 2, 64)).astype(np.float32)
        q = torch.from_numpy(x).cuda()
        ops.rope(q, None, ops.rope_frequencies(64, 1e6), win_off=dev(off), length=dev(length))
        pos = cref.positions(off, None, length, len(x))
        want, size = cref.rope(x, None, 0, cref.turns(64, 1e6), pos, False, 1.0)
        check(q, want, size, np.float32)


def test_infinities_stay_in_their_pair():
    x = np.ones((2, 2, 64), np.float16)
    x[0, 0, 5], x[1, 1, 40], x[1, 1, 63] = np.inf, np.nan, -np.inf
    q = torch.from_numpy(x).cuda()
    ops.rope(q, None, ops.rope_frequencies(48), positions=dev(np.array([3, 9], np.int32)))
    bad = ~np.isfinite(q.cpu().numpy())
    want = np.zeros_like(bad)
    want[0, 0, [5, 29]] = want[1, 1, [16, 40]] = want[1, 1, 63] = True
    assert (bad == want).all()


def test_on_a_side_stream_and_in_a_graph():
    rng = np.random.default_rng(1)
    x = rng.normal(0, 1, (9, 6, 128)).astype(np.float16)
    table, pos = ops.rope_frequencies(128), dev(np.arange(9, dtype=np.int32) * 1000)
    src = torch.from_numpy(x).cuda()
    want = ops.rope(src, None, table, positions=pos, q_out=torch.empty_like(src))[0]
    out, side = torch.zeros_like(src), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.rope(src, None, table, positions=pos, q_out=out)
    side.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.rope(src, None, table, positions=pos, q_out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        pos.add_(1)
        want = ops.rope(src, None, table, positions=pos, q_out=torch.empty_like(src))[0]


def test_refusals_of_the_python_layer():
    q = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(4, 1, 64, dtype=torch.float16, device="cuda")
    table, pos = ops.rope_frequencies(64), torch.zeros(4, dtype=torch.int32, device="cuda")
    off, ln = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (2, 1))
    for args, kw in (((q, k, table), {}), ((q, k, table), dict(positions=pos, win_off=off)),
                     ((q, k, table), dict(win_off=off)), ((q, k, table), dict(positions=pos.long())),
                     ((q, k, table), dict(positions=pos[:3])), ((q, k.float(), table), dict(positions=pos)),
                     ((q, k, table.float()), dict(positions=pos)),
                     ((q, k, ops.rope_frequencies(66)), dict(positions=pos)),
                     ((q.double(), None, table), dict(positions=pos)),
                     ((q, None, table), dict(positions=pos, k_out=k)),
                     ((q[:, :, ::2], None, table), dict(positions=pos)),
                     ((q, k, table), dict(positions=pos, q_out=q[:, :1].expand(4, 2, 64))),
                     ((q, q[:, :1], table), dict(positions=pos)),
                     ((q[0], k, table), dict(positions=pos)),
                     ((q, k, table), dict(positions=pos, q_norm=torch.ones(64))),
                     ((q, k, table), dict(win_off=off, length=ln[:0])),
                     ((q.cpu(), None, table), dict(positions=pos))):
        with pytest.raises(ops.SagerError):
            ops.rope(*args, **kw)
