"""Verification where little is left after a rejection: chunks of the vocabulary whose tokens were
all rejected, masses that are a small difference of large ones."""
import numpy as np
import pytest

import test_gpu_window as w
import window_ref as ref

pytestmark = pytest.mark.gpu

CHUNK = 4096  # logits that the kernels sum together


def struck_case(seed, n_seq, others=None, vocab=2 * CHUNK + 37, first=0, kids=2, temp=1.0):
    """Windows of a root and `kids` children that no u_accept accepts.  The children's tokens lie in
    one chunk (number `first`), whose other logits are -infinity, but for one that is `others` below
    the chunk's largest where given; three tokens of the next chunk have the larger logits."""
    rng = np.random.default_rng(seed)
    rows = 1 + kids
    x = np.full((n_seq * rows, vocab), -np.inf, np.float32)
    tok = np.zeros(n_seq * rows, np.int32)
    for s in range(n_seq):
        own = rng.choice(CHUNK, kids + 1, replace=False) + first * CHUNK
        later = rng.choice(37, 3, replace=False) + (2 if first else 1) * CHUNK
        x[s * rows, own[:kids]] = rng.uniform(3, 6, kids)
        x[s * rows, later] = rng.uniform(5, 7, 3)
        if others is not None:
            x[s * rows, own[kids]] = x[s * rows, own[:kids]].max() - others
        tok[s * rows + 1:(s + 1) * rows] = own[:kids]
        x[s * rows + 1:(s + 1) * rows, :3] = 0
    par = np.tile(np.array([-1] + [0] * kids, np.int32), n_seq)
    return dict(logits=x, tokens=tok, off=(rows * np.arange(n_seq + 1)).astype(np.int32), parent=par,
                draft=None, temp=np.full(n_seq, temp, np.float32),
                u_acc=np.full(n_seq * rows, 1 - 2.0 ** -24, np.float32),
                u_smp=np.zeros(n_seq, np.float32))


def next_of(c):
    """The kernel's and the plain form's next tokens, all paths equal and as long."""
    got = w.run_verify(c)
    want = ref.verify(c["logits"], c["tokens"], c["off"], c["parent"], c["temp"], c["u_acc"],
                      c["u_smp"], None, 16, int(np.diff(c["off"]).max()))
    np.testing.assert_array_equal(got[0], want[0])
    np.testing.assert_array_equal(got[1], want[1])
    return got[2], want[2]


def test_plain_form_of_two_rejected_tokens_in_a_chunk():
    """The example that the tests below vary: two chunks, both tokens of the first one rejected."""
    x = np.full((3, 2 * CHUNK), -np.inf, np.float32)
    x[0, 0], x[0, 1], x[0, CHUNK] = 5.75, 5.5, 6
    x[1:, 0] = 0
    c = dict(logits=x, tokens=np.array([0, 0, 1], np.int32), off=np.array([0, 3], np.int32),
             parent=np.array([-1, 0, 0], np.int32), draft=None, temp=np.ones(1, np.float32),
             u_acc=np.full(3, 0.99, np.float32), u_smp=np.zeros(1, np.float32))
    for u in (0.0, 0.5, 1 - 2.0 ** -24):
        c["u_smp"][:] = u
        got, want = next_of(c)
        assert want[0] == CHUNK and got[0] == CHUNK


@pytest.mark.parametrize("kids", [2, 3, 7])
@pytest.mark.parametrize("first,vocab", [(0, 2 * CHUNK + 37), (1, 3 * CHUNK - 5),
                                         (0, 70 * CHUNK + 1), (1, 70 * CHUNK)])
def test_verify_chunk_of_rejected_tokens_alone(kids, first, vocab):
    """Nothing is left of the chunk: no rounding makes it the last token's."""
    n = 60 if vocab < 5 * CHUNK else 6
    c = struck_case(kids + vocab, n, None, vocab, first, kids)
    for u in (0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24):
        c["u_smp"][:] = u
        got, want = next_of(c)
        np.testing.assert_array_equal(got, want)
        assert (want >= (first + 1) * CHUNK).all()


@pytest.mark.parametrize("temp", [0.25, 1.0])
@pytest.mark.parametrize("others", [8.0, 30.0, 50.0, 300.0])
def test_verify_chunk_of_rejected_tokens_and_a_small_one(others, temp):
    """What is left of the chunk is less than the rounding of its sum, and at u_sample 0 it is still
    the first token with a share."""
    c = struck_case(int(others), 60, others * temp, temp=temp)
    got, want = next_of(c)
    np.testing.assert_array_equal(got, want)
    assert (want < CHUNK).all()


# What a child may be off by once its earlier siblings are rejected, where `left` is the share that
# they leave: a row's sum by at most 31 fp64 additions after the large weight (16 a thread, 6 a
# wave, 3 a chunk, 6 over the chunks) and the share of a weight by five roundings more (the weight 2,
# its chunk's scale 1, the division and product 2): 36 2^-53 < 2^-47 of the whole, which is what the
# difference is off by: 2^-47 / left, relative.  Then prob's fp32 rounding.
def small_tol(want, left, times=1):
    return want * (w.U32 + times * 2.0 ** -47 / left) + 1e-12


@pytest.mark.parametrize("vocab", [300, 9001, 248320])
@pytest.mark.parametrize("left", [1e-2, 1e-4, 1e-6, 1e-8])
def test_verify_siblings_of_nearly_certain_tokens(left, vocab):
    """The first three children's tokens, two of them beside each other and the largest elsewhere,
    have all but `left` of the mass: the others' probabilities, given that they are rejected."""
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 1, (6, vocab)).astype(np.float32)
    big = [7, vocab - 4, vocab - 2]
    tok = np.array([0, *big, 100, 255], np.int32)
    x[:, big] = -np.inf
    for i in range(6):
        rest = np.log(np.exp(x[i].astype(np.float64)).sum() * (1 / left - 1))
        x[i, big] = rest + np.log([0.5, 0.3, 0.2])
    c = dict(logits=x, tokens=tok, off=np.array([0, 6], np.int32),
             parent=np.array([-1, 0, 0, 0, 0, 0], np.int32), draft=None, temp=np.ones(1, np.float32),
             u_acc=np.full(6, 1 - 2.0 ** -24, np.float32), u_smp=np.full(1, 0.5, np.float32))
    got = w.run_verify(c)[3]
    p, want, tol = ref.weights(x[0], 1.0), np.ones(6), np.zeros(6)
    p /= p.sum()
    for i in range(1, 6):  # (sums without what is rejected: no differences)
        want[i] = p[tok[i]] / p.sum()
        tol[i] = small_tol(want[i], p.sum())
        p[tok[i]] = 0
    assert (np.abs(got - want) <= tol).all(), (got - want) / want


@pytest.mark.parametrize("vocab", [300, 9001])
@pytest.mark.parametrize("near", [1e-2, 1e-4, 1e-6])
def test_verify_drafter_close_to_the_target(near, vocab):
    """The drafter's distribution is the target's but for `near` of each probability: what the first
    sibling's rejection leaves is that small difference."""
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 1, (3, vocab)).astype(np.float32)
    p = ref.target(x[0], 1.0)
    q = (p * (1 + near * np.where(np.arange(vocab) % 2, 1, -1))).astype(np.float32)
    rest = np.maximum(p - q.astype(np.float64), 0)
    tok = np.array([0, 10, 20], np.int32)  # (even ones have more of the target's mass)
    c = dict(logits=x, tokens=tok, off=np.array([0, 3], np.int32),
             parent=np.array([-1, 0, 0], np.int32), draft=np.stack([q, q, q]),
             temp=np.ones(1, np.float32), u_acc=np.full(3, 1 - 2.0 ** -24, np.float32),
             u_smp=np.full(1, 0.5, np.float32))
    # a second sibling that would be accepted with probability 1 says nothing: its own q is larger
    c["draft"][2] = 0
    c["draft"][2, 20] = 1
    got = w.run_verify(c, 2)[3]
    want = np.array([1.0, min(p[10] / q[10], 1), rest[20] / rest.sum()])
    # p - q is as small as `near` p, in the token's rest and in the sum of all: twice
    tol = small_tol(want, rest[20] / p[20], 2)
    assert (np.abs(got - want) <= tol).all(), (got - want) / want


@pytest.mark.parametrize("vocab", [300, 5000, 65 * CHUNK])
@pytest.mark.parametrize("left", [1e-2, 1e-5, 1e-9, 1e-11, 1e-13])
def test_verify_draw_from_what_little_is_left(left, vocab):
    """Two rejected children have all but `left` of the mass, 256 tokens share that equally: the last
    token on either side of each border between them, one step of u_sample away."""
    n = 256
    k = np.arange(1, n)
    u = np.float32(k / n)
    u = np.concatenate([np.nextafter(u, np.float32(0)), np.nextafter(u, np.float32(1))])
    x = np.full((3, vocab), -np.inf, np.float32)
    at = np.linspace(0, vocab - 3, n).astype(int) + 2
    x[0, at] = 1.0
    x[0, 1] = 1 + np.log(n * (left ** -0.5 - 1))                           # all but left ** 0.5
    x[0, 0] = 1 + np.log(n * left ** -0.5 * (left ** -0.5 - 1))            # of what it leaves too
    x[1:, 0] = 0
    got = []
    for some in np.array_split(u, 1 if vocab < 10000 else 16):
        m = len(some)
        c = dict(logits=np.tile(x, (m, 1)), tokens=np.tile(np.array([0, 0, 1], np.int32), m),
                 off=(3 * np.arange(m + 1)).astype(np.int32),
                 parent=np.tile(np.array([-1, 0, 0], np.int32), m), draft=None,
                 temp=np.ones(m, np.float32), u_acc=np.full(3 * m, 1 - 2.0 ** -24, np.float32),
                 u_smp=some)
        path, n_path, nxt, _ = w.run_verify(c)
        assert (n_path == 1).all()
        got.append(nxt)
    np.testing.assert_array_equal(np.concatenate(got), np.concatenate([at[k - 1], at[k]]))


@pytest.mark.parametrize("vocab", [300, 9001, 248320])
@pytest.mark.parametrize("lefts", [(1e-7,), (1e-7, 1e-7), (1e-3, 1e-7, 1e-8), (1e-8, 1e-4, 1e-8, 1e-7),
                                   (1e-9, 0.5), (0.5, 1e-9, 1e-9)])
def test_verify_siblings_after_nearly_certain_ones(lefts, vocab):
    """One sibling after the other leaves next to nothing of what there is: the later ones'
    probabilities are good to fp32 all the same (a difference is kept above 2^-20 of a sum that is
    good to 2^-47: 2^-26 with the token's own), and so is the last draw."""
    rng = np.random.default_rng(vocab + len(lefts))
    n = len(lefts) + 2
    e = np.exp(rng.normal(0, 1, vocab))          # weights
    own = rng.choice(np.arange(50, vocab), n, replace=False)
    if len(lefts) > 1:
        own[1] = own[0] - 1 if own[0] - 1 not in own else own[1]
    e[own[:-2]] = 0
    for i, left in reversed(list(enumerate(lefts))):
        e[own[i]] = e.sum() * (1 / left - 1)
    x = np.tile(np.log(e + (e == 0)).astype(np.float32), (n + 1, 1))
    c = dict(logits=x, tokens=np.concatenate([[0], own]).astype(np.int32),
             off=np.array([0, n + 1], np.int32), parent=np.array([-1] + [0] * n, np.int32), draft=None,
             temp=np.ones(1, np.float32), u_acc=np.full(n + 1, 1 - 2.0 ** -24, np.float32),
             u_smp=np.full(1, 0.5, np.float32))
    p, want = ref.weights(x[0], 1.0), [1.0]
    for t in own:  # (sums without what is rejected: no differences)
        want.append(p[t] / p.sum())
        p[t] = 0
    path, n_path, nxt, got = w.run_verify(c)
    want = np.array(want)
    assert (np.abs(got - want) <= want * (w.U32 + 2.0 ** -26)).all(), (got - want) / want
    accepted = want[1:] > 1 - 2.0 ** -24
    assert n_path[0] == 1 + accepted.any()
    if accepted.any():
        return
    cdf = np.cumsum(p)
    assert nxt[0] == np.nonzero(cdf > 0.5 * cdf[-1])[0][0]


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("off", [[6, 12, 0, 9, 3, 12], [0, 64, 10, 74, 5, 70], [-3, 5, 2, 1 << 30, 7]])
def test_verify_windows_that_share_rows(off, sampled):
    """Offsets that do not ascend: what the windows get is not defined, but it is their own tokens
    and paths, and the next call is what it was."""
    T = 80
    c = w.verify_case(sum(off[:3]), [T // 4] * 4, 311, branch=4, absent=True, sampled=sampled)
    base = w.run_verify(c)
    bad = dict(c, off=np.array(off, np.int32), temp=np.ones(len(off) - 1, np.float32),
               u_smp=np.full(len(off) - 1, 0.4, np.float32))
    for u in (0.0, 0.6):
        bad["u_acc"] = np.full(T, u, np.float32)
        path, n_path, nxt, _ = w.run_verify(bad, max_window=64)
        size = np.clip(np.minimum(np.array(off[1:]), T) - np.array(off[:-1]), 0, 64)
        size[(np.array(off[:-1]) < 0) | (np.array(off[:-1]) >= T)] = 0
        assert (n_path <= np.maximum(size, 0)).all() and ((n_path > 0) == (size > 0)).all()
        assert (path < np.maximum(size, 1)[:, None]).all() and (path >= -1).all()
        assert (nxt >= -1).all() and (nxt < 311).all()
    for a, b in zip(base, w.run_verify(c)):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("vocab", [2000, 20011])
def test_verify_nearly_certain_pairs_at_every_node(vocab):
    """Three windows, in whose trees every node's first two children of four have all but 1e-8."""
    rng = np.random.default_rng(vocab)
    n, n_seq = 64, 3
    par = np.array([-1] + [(i - 1) // 4 for i in range(1, n)], np.int32)
    x = rng.normal(0, 1, (n_seq * n, vocab)).astype(np.float32)
    tok = rng.integers(0, vocab, n_seq * n).astype(np.int32)
    want = np.ones(n_seq * n)
    for s in range(n_seq):
        for i in range(n):
            kids = [s * n + c for c in range(n) if par[c] == i]
            while len({tok[c] for c in kids}) < len(kids):
                tok[kids] = rng.integers(0, vocab, len(kids))
            row = x[s * n + i]
            if len(kids) > 1:
                row[tok[kids[:2]]] = -np.inf
                top = np.log(np.exp(row.astype(np.float64)).sum() * (1e8 - 1))
                row[tok[kids[:2]]] = top + np.log([0.9, 0.1])
            p = ref.weights(row, 1.0)
            for c in kids:  # (sums without what is rejected: no differences)
                want[c] = p[tok[c]] / p.sum()
                p[tok[c]] = 0
    c = dict(logits=x, tokens=tok, off=(n * np.arange(n_seq + 1)).astype(np.int32),
             parent=np.tile(par, n_seq), draft=None, temp=np.ones(n_seq, np.float32),
             u_acc=np.full(n_seq * n, 1 - 2.0 ** -24, np.float32),
             u_smp=np.full(n_seq, 0.5, np.float32))
    got = w.run_verify(c)[3]
    assert (np.abs(got - want) <= want * (w.U32 + 2.0 ** -26)).all(), np.abs(got / want - 1).max()
