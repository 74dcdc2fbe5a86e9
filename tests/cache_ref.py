"""Plain 64-bit forms (numpy, on the CPU) of rotary positions, the quantised cache and the sliding
attention, and inputs for them."""
import numpy as np

import window_ref as ref


def positions(off, parent, length, n_tokens, max_window=64):
    """Each row's position in its sequence, -1 for rows without one."""
    pos = -np.ones(n_tokens, np.int64)
    for s in range(len(off) - 1):
        if parent is None:
            n = int(off[s + 1] - off[s])
            pos[off[s]:off[s + 1]] = length[s] + np.arange(n)
            continue
        up = ref.up_of(parent, off, s, max_window)
        for i in range(len(up)):
            line = ref.line_of(up, i)
            if line:
                pos[off[s] + i] = length[s] + len(line) - 1
    return pos


def turns(rot, base, kind=None, factor=1.0, trained=0, slow=1.0, fast=32.0):
    f = base ** (-np.arange(0, rot, 2) / rot) / (2 * np.pi)
    i = np.arange(rot // 2)
    if kind == "linear":
        return f / factor
    if kind == "yarn":
        lo, hi = (rot * np.log(trained / (t * 2 * np.pi)) / (2 * np.log(base)) for t in (fast, slow))
        lo, hi = max(np.floor(lo), 0), min(np.ceil(hi), rot - 1)
        r = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * r + f * (1 - r)
    if kind == "by_turns":
        g = np.clip((trained * f - slow) / (fast - slow), 0, 1)
        return (1 - g) * f / factor + g * f
    return f


def rope(x, w, eps, table, pos, neighbours, mscale):
    """x [n, heads, dim] -> (y, size): size bounds what a relative error of the parts moves."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(2, keepdims=True) + eps) * w.astype(np.float64)
    rot = 2 * len(table)
    turn = pos[:, None] * table
    a = 2 * np.pi * (turn - np.rint(turn))
    c, s = np.cos(a)[:, None] * mscale, np.sin(a)[:, None] * mscale
    i, j = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if neighbours else \
        (np.arange(rot // 2), np.arange(rot // 2, rot))
    y, size = x.copy(), np.abs(x)
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    size[..., i] = size[..., j] = (np.abs(x[..., i]) + np.abs(x[..., j])) * mscale
    return y, size


def quantise(x):
    """fp16 [..., dim] -> (codes int8, scales fp16 [..., dim / 32])."""
    g = x.astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        top = np.abs(g).max(-1)
        d = np.minimum((top / 127).astype(np.float16), np.float16(515.5))
        odd = ~np.isfinite(top)
        d = np.where(odd, np.float16(np.nan), d)
        step = np.where(odd | (d == 0), 1, d).astype(np.float64)[..., None]
        code = np.clip(np.rint(g / step), -127, 127)
        code = np.where((odd | (d == 0))[..., None], 0, code)
    return code.astype(np.int8).reshape(x.shape), d


def values(code, scale):
    g = code.astype(np.float64).reshape(*code.shape[:-1], -1, 32)
    return (g * scale.astype(np.float64)[..., None]).reshape(code.shape)


def attention(q, k, v, kc, vc, pages, length, off, parent, scale, page_size, out, reach=0, sinks=0,
              max_window=64):
    """kc, vc: [pages, heads, slots, dim] as values.  Returns (out, spread): out fp64 with absent
    nodes' rows 0 and rows behind the windows as given; spread = sum p |v|."""
    out = out.astype(np.float64).copy()
    spread = np.zeros_like(out)
    heads, n_kv = q.shape[1], k.shape[1]
    G, n_pages, far = heads // n_kv, kc.shape[0], reach or 1 << 40
    for s in range(len(off) - 1):
        if parent is None:
            size = min(int(off[s + 1] - off[s]), max_window)
            lines = [list(range(i + 1)) for i in range(size)]
        else:
            up = ref.up_of(parent, off, s, max_window)
            lines = [sorted(ref.line_of(up, i)) for i in range(len(up))]
        n = max(0, min(int(length[s]), pages.shape[1] * page_size))
        j = np.arange(n)
        pg = pages[s, j // page_size]
        j = j[(pg >= 0) & (pg < n_pages)]
        pg, sl = pages[s, j // page_size], j % page_size
        for i, line in enumerate(lines):
            row = off[s] + i
            if not line:
                out[row] = 0
                continue
            me = n + len(line) - 1
            see = (j < sinks) | (j > me - far)
            seen = np.array([m for d, m in enumerate(line) if n + d < sinks or n + d > me - far],
                            int) + off[s]
            for h in range(heads):
                g = h // G
                K = np.concatenate([kc[pg[see], g, sl[see]], k[seen, g]]).astype(np.float64)
                V = np.concatenate([vc[pg[see], g, sl[see]], v[seen, g]]).astype(np.float64)
                with np.errstate(invalid="ignore"):
                    x = K @ q[row, h].astype(np.float64) * scale
                    e = np.exp(x - x.max())
                    out[row, h] = e @ V / e.sum()
                    spread[row, h] = e @ np.abs(V) / e.sum()
    return out, spread
