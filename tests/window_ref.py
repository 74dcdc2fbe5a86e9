"""Plain 64-bit forms (numpy, on the CPU) of the verify window's operators,
and inputs for them."""
import numpy as np

REST = 2.0 ** -30


def off_of(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)


def up_of(parent, off, s, max_window=64):
    """Parents of a window's nodes: -1 for the root, None for absent ones."""
    n = min(int(off[s + 1] - off[s]), max_window)
    up = []
    for i in range(n):
        p = i - 1 if parent is None else int(parent[off[s] + i])
        ok = i == 0 or (0 <= p < i and up[p] is not None)
        up.append(None if not ok else -1 if i == 0 else p)
    return up


def line_of(up, i):
    """Node i and its ancestors; [] if it is absent."""
    if up[i] is None:
        return []
    line = [i]
    while i > 0:
        i = up[i]
        line.append(i)
    return line


def attention(q, k, v, kc, vc, pages, length, off, parent, scale, page_size, out, max_window=64):
    """Returns (out, spread): out fp64 with absent nodes' rows 0 and rows behind the windows as
    given; spread = sum p |v| (what a relative error of p moves)."""
    out = out.astype(np.float64).copy()
    spread = np.zeros_like(out)
    heads, n_kv = q.shape[1], k.shape[1]
    G, n_pages = heads // n_kv, kc.shape[0]
    for s in range(len(off) - 1):
        up = up_of(parent, off, s, max_window)
        n = max(0, min(int(length[s]), pages.shape[1] * page_size))
        at = [(pages[s, j // page_size], j % page_size) for j in range(n)]
        at = [(p, t) for p, t in at if 0 <= p < n_pages]
        pg, sl = (np.array([x[i] for x in at], dtype=int) for i in (0, 1))
        for i in range(len(up)):
            row, line = off[s] + i, line_of(up, i)
            if not line:
                out[row] = 0
                continue
            seen = off[s] + np.array(sorted(line))
            for h in range(heads):
                g = h // G
                K = np.concatenate([kc[pg, g, sl], k[seen, g]]).astype(np.float64)
                V = np.concatenate([vc[pg, g, sl], v[seen, g]]).astype(np.float64)
                x = K @ q[row, h].astype(np.float64) * scale
                e = np.exp(x - x.max())
                out[row, h] = e @ V / e.sum()
                with np.errstate(invalid="ignore"):
                    spread[row, h] = e @ np.abs(V) / e.sum()
    return out, spread


def weights(logits, t):
    """The target's probabilities of a row times a number that keeps equal logits' weights exact (all
    0 if nothing is left)."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    m = x.max()
    if m == -np.inf:
        return np.zeros_like(x)
    if not t > 0:
        r = np.zeros_like(x)
        r[np.argmax(x)] = 1
        return r
    with np.errstate(invalid="ignore"):
        return np.where(x == m, 1.0, np.where(x - m == -np.inf, 0.0, np.exp((x - m) / np.float64(t))))


def target(logits, t):
    e = weights(logits, t)
    return e / e.sum() if e.any() else e


def verify(logits, tokens, off, parent, temp, u_acc, u_smp, draft=None, max_children=16,
           max_window=64, prob=None):
    n_seq, V = len(off) - 1, logits.shape[1]
    path = -np.ones((n_seq, max_window), np.int32)
    n_path, nxt = np.zeros(n_seq, np.int32), -np.ones(n_seq, np.int32)
    prob = np.zeros(len(tokens)) if prob is None else prob.astype(np.float64).copy()
    for s in range(n_seq):
        raw = up_of(parent, off, s, max_window)
        edge = [i - 1 if parent is None else int(parent[off[s] + i]) for i in range(len(raw))]
        up = []
        for i, p in enumerate(raw):  # children past max_children are absent too
            if i > 0 and p is not None:
                rank = sum(edge[j] == p for j in range(1, i))
                if up[p] is None or (draft is not None and rank >= max_children):
                    p = None
            up.append(p)
        if not up:
            continue
        rest, taken = {}, {}
        for i in range(len(up)):
            prob[off[s] + i] = 1.0 if i == 0 else 0.0
        for i in range(len(up)):
            if up[i] is None:
                continue
            e = weights(logits[off[s] + i], temp[s])
            r = e / e.sum() if e.any() else e
            S = 1.0 if r.sum() > 0 else 0.0
            for c in range(i + 1, len(up)):
                if up[c] != i:
                    continue
                row, tok = off[s] + c, int(tokens[off[s] + c])
                real = 0 <= tok < V
                q = None if draft is None else draft[row].astype(np.float64)
                rc = r[tok] if real else 0.0
                qc = (q[tok] if q is not None else 1.0) if real else (0.0 if q is not None else 1.0)
                bar = qc * S
                prob[row] = (1.0 if rc > 0 else 0.0) if rc >= bar else rc / bar
                if i not in taken and float(u_acc[row]) * bar < rc:
                    taken[i] = c
                if q is None:
                    left = S - rc
                    if left >= REST * S and real:
                        r, e = r.copy(), e.copy()
                        r[tok] = e[tok] = 0
                        S = left
                else:
                    new = np.maximum((r / S if S > 0 else r * 0) - q, 0)
                    if new.sum() >= REST:
                        r, S, e = new, new.sum(), new
            rest[i] = e  # (drawn from without a division: borders of equal weights stay exact)
        at, n = 0, 0
        while True:
            path[s, n] = at
            n += 1
            if at not in taken:
                break
            at = taken[at]
        n_path[s] = n
        r = rest[at]
        if r.sum() > 0:
            cdf = np.cumsum(r)
            hit = np.nonzero((cdf > np.float64(u_smp[s]) * cdf[-1]) & (r > 0))[0]
            nxt[s] = hit[0] if len(hit) else np.nonzero(r)[0][-1]
    return path, n_path, nxt, prob


def tree(rng, n, branch, absent=False):
    """Parents of a window of n nodes, at most `branch` children a node."""
    par, kids = [-1], [0] * n
    for i in range(1, n):
        free = [p for p in range(i) if kids[p] < branch and i - p <= 2 * branch + 1] or [i - 1]
        p = int(rng.choice(free))
        kids[p] += 1
        par.append(p)
    if absent:
        for i in range(3, n, 4):
            par[i] = int(rng.choice([-1, i, i + 3, -7, 1 << 30]))
    return par[:n]
