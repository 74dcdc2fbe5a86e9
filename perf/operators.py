"""The operators of a verify window, as cases that can be timed.

A session that decodes speculatively runs a window of tokens a step: the last
token and a chain or a tree of drafts.  Between the library's projections,
its MoE layer and its LM head lie four operators, one kind of case each:

  norm    the residual's addition, the RMS norm and the Q8_K of the normed
          rows that the next projections (or the MoE layer) take.
  attn    the window's attention over a paged cache and over the window's own
          ancestors.
  verify  which drafts the target's probabilities accept, and the token that
          follows them, from given random numbers.
  commit  the accepted tokens' keys and values written behind the cache.

Each case runs one operator: in its plain form, elementary torch operations
(`own` false), or by the library's entry point (`own` true).
"""
import math

import torch

own = False

DEVICE = "cuda"
QK = 256           # values of a Q8_K block
Q8K_BYTES = 276    # fp32 d | 256 int8 | 8 int16
# less than this share of the mass left after a rejected draft counts as none
REST = 2.0 ** -30


def listed():
    return [
        # a verify window of one token and three drafts, after the output projection
        {"name": "norm_t4_f16", "kind": "norm", "rows": 4, "hidden": 2048, "dtype": "f16",
         "add": True, "out": "both"},
        # a prompt's ragged last chunk on fp32 buffers, only the Q8_K is used
        {"name": "norm_t509_f32", "kind": "norm", "rows": 509, "hidden": 1280, "dtype": "f32",
         "add": True, "out": "q8"},
        # a long prefill chunk
        {"name": "norm_t4096_f16", "kind": "norm", "rows": 4096, "hidden": 2048, "dtype": "f16",
         "add": True, "out": "both"},
        # the chain of a token and three drafts over one sequence's cache
        {"name": "attn_chain4_4k", "kind": "attn", "seqs": 1, "window": 4, "ragged": False,
         "branch": 1, "absent": False, "pad": 0, "kv_heads": 2, "group": 8, "dim": 256,
         "len_lo": 4099, "len_hi": 4099, "page": 64},
        # sequences decoded together without drafts, one token each
        {"name": "attn_t1_batch", "kind": "attn", "seqs": 24, "window": 1, "ragged": False,
         "branch": 1, "absent": False, "pad": 0, "kv_heads": 8, "group": 4, "dim": 128,
         "len_lo": 77, "len_hi": 4001, "page": 16},
        # ragged trees of a padded batch, three query heads a kv head, a sequence with an empty cache
        {"name": "attn_tree_batch", "kind": "attn", "seqs": 7, "window": 13, "ragged": True,
         "branch": 3, "absent": True, "pad": 5, "kv_heads": 5, "group": 3, "dim": 64,
         "len_lo": 0, "len_hi": 9001, "page": 32},
        # a wide tree over a long context: the largest
        {"name": "attn_tree64_128k", "kind": "attn", "seqs": 1, "window": 64, "ragged": False,
         "branch": 4, "absent": False, "pad": 0, "kv_heads": 2, "group": 8, "dim": 256,
         "len_lo": 131071, "len_hi": 131071, "page": 256},
        # the window of three greedy drafts against the model's vocabulary
        {"name": "verify_chain4", "kind": "verify", "seqs": 1, "window": 4, "ragged": False,
         "branch": 1, "absent": False, "pad": 0, "vocab": 248320, "sampled": False},
        # a batch of sampled trees with the drafter's distributions, temperatures from 0 up
        {"name": "verify_sampled", "kind": "verify", "seqs": 6, "window": 7, "ragged": True,
         "branch": 2, "absent": True, "pad": 3, "vocab": 50257, "sampled": True},
        # one wide tree, the largest vocabulary
        {"name": "verify_tree64", "kind": "verify", "seqs": 1, "window": 64, "ragged": False,
         "branch": 4, "absent": False, "pad": 0, "vocab": 248320, "sampled": False},
        # the accepted part of a window of four behind one sequence's cache, ten attention layers
        {"name": "commit_t4_l10", "kind": "commit", "seqs": 1, "window": 4, "ragged": False,
         "layers": 10, "kv_heads": 2, "dim": 256, "len_lo": 4099, "len_hi": 4099, "page": 64},
        # the same for a batch of trees
        {"name": "commit_batch_l40", "kind": "commit", "seqs": 32, "window": 16, "ragged": True,
         "layers": 40, "kv_heads": 8, "dim": 128, "len_lo": 0, "len_hi": 1000, "page": 16},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "attn", "attn", "verify", "verify", "commit"])
    if kind == "norm":
        hidden = QK * _log_int(rng, 1, 32)
        most = max(1, 4096 * 2048 // hidden)
        return {"kind": kind, "rows": _log_int(rng, 1, min(4096, most)), "hidden": hidden,
                "dtype": rng.choice(["f16", "f16", "f32"]), "add": rng.random() < 0.7,
                "out": rng.choice(["both", "q8", "normed"])}
    seqs = _log_int(rng, 1, 32)
    if kind == "commit":
        lo = rng.choice([0, 13, _log_int(rng, 1, 1000)])
        return {"kind": kind, "seqs": seqs, "window": _log_int(rng, 1, 16),
                "ragged": rng.random() < 0.5, "layers": _log_int(rng, 1, 40),
                "kv_heads": rng.randint(1, 8), "dim": rng.choice([64, 128]),
                "len_lo": lo, "len_hi": lo + _log_int(rng, 1, 1000),
                "page": rng.choice([16, 32, 64])}
    branch = rng.choice([1, 1, 2, 3, 5])
    tree = {"seqs": seqs, "ragged": seqs > 1 and rng.random() < 0.6, "branch": branch,
            "absent": branch > 1 and rng.random() < 0.4, "pad": rng.choice([0, 0, 1, 9])}
    if kind == "verify":
        sampled = rng.random() < 0.5
        vocab = _log_int(rng, 1000, 248320)
        rows = max(1, min(64 * 248320, 16 * 2 ** 20 if sampled else 2 ** 24) // vocab)
        window = _log_int(rng, 1, max(1, min(64, rows // seqs)))
        return {"kind": kind, **tree, "window": window, "vocab": vocab, "sampled": sampled}
    dim = rng.choice([64, 128, 128, 256])
    kv_heads, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16])
    window = _log_int(rng, 1, 64)
    # the largest listed case reads 1.3e8 values of keys and values and has 7e10 products
    most = min(1.3e8 / (2 * seqs * kv_heads * dim),
               7e10 / (2 * seqs * window * kv_heads * group * dim), 131072)
    hi = _log_int(rng, 1, max(2, int(most)))
    return {"kind": kind, **tree, "window": window, "kv_heads": kv_heads, "group": group,
            "dim": dim, "len_lo": rng.choice([0, hi, _log_int(rng, 1, hi) if hi > 1 else 1]),
            "len_hi": hi, "page": rng.choice([16, 32, 64, 128, 256])}


# ---- inputs -------------------------------------------------------------------

def _generator(seed, salt):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed * 1000003 + salt)
    return g


def _normal(gen, *shape, scale=1.0, dtype=torch.float16):
    return (torch.randn(shape, device=DEVICE, generator=gen) * scale).to(dtype)


def _windows(case):
    """The windows' sizes: whole windows, or sizes from 1 up to the largest."""
    n, most = case["seqs"], case["window"]
    if not case["ragged"]:
        return [most] * n
    return [1 + (i * 7 + most - 1) % most for i in range(n)]


def _lengths(case):
    """The caches' lengths, from the shortest to the longest."""
    n, lo, hi = case["seqs"], case["len_lo"], case["len_hi"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _offsets(sizes):
    off = [0]
    for s in sizes:
        off.append(off[-1] + s)
    return off


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEVICE)


def _parents(case, sizes):
    """Node i of a window hangs on node (i - 1) // branch; where nodes are absent, every fifth
    (and with it what hangs on it) has no parent."""
    par = []
    for s in sizes:
        par += [-1 if i == 0 or (case["absent"] and i % 5 == 4) else (i - 1) // case["branch"]
                for i in range(s)]
    return par + [-1] * case["pad"]


def _pages(case, gen, lengths, more=0):
    """A table of pages in the pool's random order; entries past a sequence's last page are -1."""
    per_seq = max(1, max((n + more + case["page"] - 1) // case["page"] for n in lengths))
    used = [(n + more + case["page"] - 1) // case["page"] for n in lengths]
    n_pages = sum(used) + 3
    order = torch.randperm(n_pages, generator=gen, device=DEVICE).to(torch.int32)
    table, at = torch.full((len(lengths), per_seq), -1, dtype=torch.int32, device=DEVICE), 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    return table, n_pages


def _prepare_norm(case, seed):
    gen = _generator(seed, 1)
    dt = torch.float16 if case["dtype"] == "f16" else torch.float32
    n, h = case["rows"], case["hidden"]
    x = _normal(gen, n, h, scale=2.0, dtype=dt)
    x[:, 5::97] *= 8  # a few channels of a residual stream are far larger than the rest
    return {"x": x, "y": _normal(gen, n, h, dtype=dt) if case["add"] else None,
            "w": 1 + 0.2 * torch.randn(h, device=DEVICE, generator=gen), "eps": 1e-6}


def _prepare_attn(case, seed):
    gen = _generator(seed, 2)
    sizes, lengths = _windows(case), _lengths(case)
    off = _offsets(sizes)
    T, H, G, D = off[-1] + case["pad"], case["kv_heads"], case["group"], case["dim"]
    pages, n_pages = _pages(case, gen, lengths)
    shape = (1, n_pages, H, case["page"], D)
    # q, k and v of the window are slices of one projection's output
    qkv = _normal(gen, T, (H * G + 2 * H) * D)
    q, k, v = qkv.split([H * G * D, H * D, H * D], dim=1)
    q.mul_(2.0)
    return {"q": q.view(T, H * G, D), "k": k.view(T, H, D), "v": v.view(T, H, D),
            "k_cache": _normal(gen, *shape), "v_cache": _normal(gen, *shape),
            "pages": pages, "length": _ints(lengths), "win_off": _ints(off),
            "parent": _ints(_parents(case, sizes)), "scale": 1 / math.sqrt(D),
            "out": torch.zeros((T, H * G, D), dtype=torch.float16, device=DEVICE)}


def _prepare_verify(case, seed):
    gen = _generator(seed, 3)
    sizes = _windows(case)
    off = _offsets(sizes)
    T, V, n = off[-1] + case["pad"], case["vocab"], case["seqs"]
    par = _parents(case, sizes)
    # logits with a few likely tokens a row over a long tail
    logits = _normal(gen, T, V, scale=2.0, dtype=torch.float32)
    at = torch.randint(V, (T, 24), device=DEVICE, generator=gen)
    logits.scatter_add_(1, at, 6 + 6 * torch.rand((T, 24), device=DEVICE, generator=gen))
    temp = _ints([(0.8, 1.0, 0.0, 1.3)[i % 4] for i in range(n)], torch.float32)
    # the drafter: its distribution of a node's token is near the target's at the parent
    start = [o for o, s in zip(off, sizes) for _ in range(s)] + [0] * case["pad"]
    row = _ints([s + max(p, 0) for s, p in zip(start, par)], torch.int64)
    guess = logits[row] + 0.5 * torch.randn((T, V), device=DEVICE, generator=gen)
    q = torch.softmax(guess, 1)
    tokens = (q / torch.empty_like(q).exponential_(generator=gen)).argmax(1).to(torch.int32)
    return {"logits": logits, "tokens": tokens, "win_off": _ints(off), "parent": _ints(par),
            "temperature": temp, "draft_probs": q if case["sampled"] else None,
            "u_accept": torch.rand(T, device=DEVICE, generator=gen),
            "u_sample": torch.rand(n, device=DEVICE, generator=gen)}


def _prepare_commit(case, seed):
    gen = _generator(seed, 4)
    sizes, lengths = _windows(case), _lengths(case)
    off = _offsets(sizes)
    T, L, H, D, n, W = off[-1], case["layers"], case["kv_heads"], case["dim"], case["seqs"], \
        case["window"]
    pages, n_pages = _pages(case, gen, lengths, more=W)
    # accepted paths as a verification leaves them: the root and some of its descendants, in order
    size = _ints(sizes, torch.int64)
    keep = torch.rand((n, W), device=DEVICE, generator=gen) < 0.7
    node = torch.arange(W, device=DEVICE)
    keep = (keep | (node == 0)) & (node < size[:, None])
    path = torch.where(keep, node, W).sort(1).values
    return {"k": _normal(gen, L, T, H, D), "v": _normal(gen, L, T, H, D),
            "k_cache": _normal(gen, L, n_pages, H, case["page"], D),
            "v_cache": _normal(gen, L, n_pages, H, case["page"], D),
            "pages": pages, "length": _ints(lengths), "win_off": _ints(off),
            "path": torch.where(path < W, path, -1).to(torch.int32),
            "n_path": keep.sum(1).to(torch.int32)}


def prepare(case, seed):
    state = {"norm": _prepare_norm, "attn": _prepare_attn, "verify": _prepare_verify,
             "commit": _prepare_commit}[case["kind"]](case, seed)
    state["case"] = case
    if own:
        _handles(case, state)
    return state


def _handles(case, state):
    """What a program keeps for the library's calls: output buffers, objects with workspaces."""
    from sager_amd import ops
    if case["kind"] == "norm":
        x = state["x"]
        n, h = x.shape
        state["x_out"] = torch.empty_like(x) if case["add"] else None
        state["xn"] = torch.empty_like(x) if case["out"] != "q8" else None
        state["xq"] = ops.q8k_empty(n, h) if case["out"] != "normed" else None
        state["values"] = torch.empty((n, h // QK, QK), dtype=torch.float16, device=DEVICE)
    elif case["kind"] == "verify":
        state["verify"] = ops.TreeVerify(
            case["vocab"], max_tokens=state["logits"].shape[0], max_seqs=case["seqs"],
            max_window=case["window"], max_children=case["branch"] if case["sampled"] else 0)
        state["prob"] = torch.zeros(state["logits"].shape[0], device=DEVICE)
    else:
        state["cache"] = ops.KvCache(state["k_cache"], state["v_cache"], state["pages"],
                                     state["length"])
        if case["kind"] == "attn":
            state["attn"] = ops.TreeAttention(
                case["kv_heads"] * case["group"], case["kv_heads"], case["dim"],
                max_tokens=state["q"].shape[0], max_seqs=case["seqs"],
                max_window=case["window"], max_len=case["len_hi"])


# ---- the plain forms ------------------------------------------------------------

def _plain_norm(state):
    x, out = state["x"], state["case"]["out"]
    r = x if state["y"] is None else (x.float() + state["y"].float()).to(x.dtype)
    f = r.float()
    xn = (f * torch.rsqrt((f * f).mean(1, keepdim=True) + state["eps"]) * state["w"]).to(x.dtype)
    got = {} if state["y"] is None else {"x_out": r}
    if out != "q8":
        got["xn"] = xn
    if out != "normed":
        b = xn.float().view(x.shape[0], -1, QK)
        d = b.abs().amax(2, keepdim=True).clamp_min(1e-30) / 127
        # the codes as the values that they stand for, in the activations' 16 bits
        got["values"] = ((b / d).round().clamp(-127, 127) * d).half()
    return got


def _tree(state, window):
    """Rows of the windows' nodes [n, W], which of them there are, and who is whose ancestor
    (or the node itself) [n, W, W]; a node that does not hang on its window's first is absent."""
    off = state["win_off"].long()
    node = torch.arange(window, device=off.device)
    row = off[:-1, None] + node
    there = row < off[1:, None]
    row = torch.where(there, row, 0)
    par = torch.where(there, state["parent"].long()[row], -1)
    edge = (par >= 0) & (par < node) & (node > 0)
    up = (node[:, None] == node) | (edge[:, :, None] & (par[:, :, None] == node))
    up = up.float()
    for _ in range(max(1, (window - 1).bit_length())):
        up = (up @ up).clamp_max(1)
    there = there & (up[:, :, 0] > 0)
    return row, there, (up > 0) & there[:, :, None]


def _plain_attn(state):
    case = state["case"]
    n, W, H, G, D = (case[c] for c in ("seqs", "window", "kv_heads", "group", "dim"))
    row, there, up = _tree(state, W)
    page, pages = case["page"], state["pages"].long()
    pos = torch.arange(pages.shape[1] * page, device=pages.device)[:case["len_hi"]]
    at = pages[:, pos // page]
    seen = (pos < state["length"][:, None]) & (at >= 0)
    at = at.clamp_min(0)
    head = torch.arange(H, device=pages.device)

    def cached(c):  # [n, H, len, D]
        return c[0][at[:, None, :], head[None, :, None], (pos % page)[None, None, :]].float()

    q = state["q"][row].float().view(n, W, H, G, D).permute(0, 2, 1, 3, 4).reshape(n, H, W * G, D)
    k_new = state["k"][row].float().transpose(1, 2).contiguous()
    v_new = state["v"][row].float().transpose(1, 2).contiguous()
    k = torch.cat([cached(state["k_cache"]), k_new], 2)
    s = q @ k.transpose(2, 3).contiguous() * state["scale"]
    mask = torch.cat([seen[:, None, :].expand(n, W, -1), up], 2)
    mask = (mask & there[:, :, None]).repeat_interleave(G, 1)[:, None]
    s = s.masked_fill(~mask, -math.inf)
    top = s.amax(3, keepdim=True)
    e = torch.exp(s - torch.where(top > -math.inf, top, 0))
    v = torch.cat([cached(state["v_cache"]), v_new], 2)
    total = e.sum(3, keepdim=True)
    o = e @ v / torch.where(total > 0, total, 1)
    o = o.view(n, H, W, G, D).permute(0, 2, 1, 3, 4).reshape(n, W, H * G, D).half()
    # (past a window's end, its first row once more)
    node = torch.arange(W, device=row.device)
    off = state["win_off"].long()
    node = torch.where(node < (off[1:] - off[:-1])[:, None], node, 0)
    state["out"][off[:-1, None] + node] = o[torch.arange(n, device=row.device)[:, None], node]
    return {"out": state["out"]}


def _plain_verify(state):
    case = state["case"]
    n, W, V = case["seqs"], case["window"], case["vocab"]
    logits, dev = state["logits"], state["logits"].device
    T = logits.shape[0]
    # per row: its sequence, its parent's row (itself where it has none), whether it is in a tree
    off, at = state["win_off"].long(), torch.arange(T, device=dev)
    seq = torch.searchsorted(off[1:], at, right=True).clamp_max(n - 1)
    start, par = off[seq], state["parent"].long()
    edge = (at < off[-1]) & (at > start) & (par >= 0) & (start + par < at)
    up = torch.where(edge, start + par, at)
    root = up
    for _ in range(max(1, (W - 1).bit_length())):
        root = root[root]
    up = torch.where(edge & (root == start), up, -1)
    token = state["tokens"].long()
    sib = (up[:, None] == up) & (up >= 0)[:, None]
    rank = torch.tril(sib, -1).sum(1)
    # the target's probabilities; temperature 0 puts all on the likeliest token
    t = state["temperature"].double()[seq][:, None]
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(1, keepdim=True)
    some = top > -math.inf
    z = torch.where(x == top, 0.0, x - top)
    R = torch.where(some, torch.exp(z / torch.where(t > 0, t, 1)), 0)
    first = torch.where(x == top, torch.arange(V, device=dev), V).amin(1, keepdim=True)
    greedy = (torch.arange(V, device=dev) == first) & some
    R = torch.where(t > 0, R, greedy.double())
    del x, z, greedy
    S = R.sum(1)
    R /= torch.where(S > 0, S, 1)[:, None]
    S = (S > 0).double()
    prob = torch.zeros(T, dtype=torch.float64, device=dev)
    prob[off[:-1]] = 1
    taken = torch.full((T,), -1, dtype=torch.long, device=dev)
    u = state["u_accept"].double()
    for j in range(case["branch"]):  # the children of rank j, all at once
        c = torch.nonzero((up >= 0) & (rank == j))[:, 0]
        p, tok = up[c], token[c]
        r = R[p, tok]
        q = state["draft_probs"][c].double() if case["sampled"] else None
        qc = q.gather(1, tok[:, None])[:, 0] if case["sampled"] else torch.ones_like(r)
        # (what is left in R is what a rejection of all children of lower rank leaves)
        ok = u[c] * qc * S[p] < r
        prob[c] = torch.where(r >= qc * S[p], (r > 0).double(), r / (qc * S[p]))
        taken[p] = torch.where((taken[p] < 0) & ok, c, taken[p])
        if case["sampled"]:
            rest = (R[p] / torch.where(S[p] > 0, S[p], 1)[:, None] - q).clamp_min(0)
            left = rest.sum(1)
            keep = left >= REST
            R[p] = torch.where(keep[:, None], rest, R[p])
            S[p] = torch.where(keep, left, S[p])
        else:
            left = S[p] - r
            keep = left >= REST * S[p]
            R[p, tok] = torch.where(keep, 0, r)
            S[p] = torch.where(keep, left, S[p])
    cur = off[:-1]
    end, base = cur, cur
    path = torch.full((n, W), -1, dtype=torch.int32, device=dev)
    n_path = torch.zeros(n, dtype=torch.int32, device=dev)
    for i in range(W):
        path[:, i] = torch.where(cur >= 0, cur - base, -1)
        n_path += cur >= 0
        end = torch.where(cur >= 0, cur, end)
        cur = torch.where(cur >= 0, taken[cur.clamp_min(0)], -1)
    cdf = R[end].cumsum(1)
    goal = state["u_sample"].double()[:, None] * cdf[:, -1:]
    nxt = (cdf <= goal).sum(1)
    last = torch.where(R[end] > 0, torch.arange(V, device=dev), -1).amax(1)
    return {"path": path, "n_path": n_path, "next": torch.minimum(nxt, last).to(torch.int32),
            "prob": prob.float()}


def _plain_commit(state):
    case = state["case"]
    page, W = case["page"], case["window"]
    node = torch.arange(W, device=state["path"].device)
    # (past a path's end, its first row once more)
    i = torch.where(node < state["n_path"][:, None], node, 0)
    row = (state["win_off"].long()[:-1, None] + state["path"].long().gather(1, i)).view(-1)
    pos = state["length"].long()[:, None] + i
    at = state["pages"].long().gather(1, pos // page).view(-1)
    pos = pos.view(-1)
    head = torch.arange(case["kv_heads"], device=at.device)
    for name in ("k", "v"):
        state[name + "_cache"][:, at[:, None], head, (pos % page)[:, None]] = state[name][:, row]
    return {"k": state["k_cache"], "v": state["v_cache"],
            "length": state["length"] + state["n_path"]}


# ---- the library's calls --------------------------------------------------------

def _own(state):
    from sager_amd import ops
    case = state["case"]
    if case["kind"] == "norm":
        ops.add_rmsnorm_q8_k(state["x"], state["w"], state["eps"], y=state["y"],
                             x_out=state["x_out"], xn=state["xn"], xq=state["xq"])
        got = {} if state["y"] is None else {"x_out": state["x_out"]}
        if state["xn"] is not None:
            got["xn"] = state["xn"]
        if state["xq"] is not None:
            b = state["xq"].view(state["x"].shape[0], -1, Q8K_BYTES)
            got["values"] = torch.mul(b[:, :, 4:4 + QK].view(torch.int8),
                                      b.view(torch.float32)[:, :, :1], out=state["values"])
        return got
    if case["kind"] == "attn":
        return {"out": state["attn"].forward(
            state["q"], state["k"], state["v"], state["cache"], state["win_off"],
            state["parent"], scale=state["scale"], out=state["out"])}
    if case["kind"] == "verify":
        path, n_path, nxt, prob = state["verify"].forward(
            state["logits"], state["tokens"], state["win_off"], state["parent"],
            state["temperature"], state["u_accept"], state["u_sample"],
            draft_probs=state["draft_probs"], prob=state["prob"])
        return {"path": path, "n_path": n_path, "next": nxt, "prob": prob}
    length = state["cache"].commit(state["k"], state["v"], state["win_off"], state["path"],
                                   state["n_path"])
    return {"k": state["k_cache"], "v": state["v_cache"], "length": length}


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "attn": _plain_attn, "verify": _plain_verify,
            "commit": _plain_commit}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, h = case["rows"], case["hidden"]
        el = 2 if case["dtype"] == "f16" else 4
        streams = (3 if case["add"] else 1) + (1 if case["out"] != "q8" else 0)
        q8 = n * h * Q8K_BYTES / QK if case["out"] != "normed" else 0
        return {"bytes": n * h * el * streams + 4 * h + q8, "flops": 8.0 * n * h}
    sizes = _windows(case)
    if kind == "verify":
        rows = sum(sizes)
        return {"bytes": 4.0 * rows * case["vocab"] * (2 if case["sampled"] else 1),
                "flops": 10.0 * rows * case["vocab"]}
    H, D = case["kv_heads"], case["dim"]
    if kind == "commit":
        rows = sum(1 + 0.7 * (s - 1) for s in sizes)
        return {"bytes": case["layers"] * rows * H * D * 8.0, "flops": 0}
    total = flops = 0
    for s, n in zip(sizes, _lengths(case)):
        total += 4.0 * (n + s) * H * D + 4.0 * s * H * case["group"] * D
        flops += 4.0 * s * H * case["group"] * D * (n + s / 2)
    return {"bytes": total, "flops": flops}


# ---- the same in 64 bits ----------------------------------------------------------

def _exact_norm(case, s):
    x, y, w = s["x"].double(), s["y"], s["w"].double()
    total = x if y is None else x + y.double()
    r = total.to(s["x"].dtype).double()  # the residual is what is stored
    normed = r / (r.pow(2).sum(1) / r.shape[1] + s["eps"]).sqrt()[:, None] * w
    got = {} if y is None else {"x_out": total}
    if case["out"] != "q8":
        got["xn"] = normed
    if case["out"] != "normed":
        b = normed.to(s["x"].dtype).double().reshape(r.shape[0], -1, QK)
        step = b.abs().max(2)[0][:, :, None] / 127
        got["values"] = torch.round(b / step) * step
    return got


def _exact_attn(case, s):
    """One sequence and one kv head after the other."""
    off, par, G = s["win_off"].tolist(), s["parent"].tolist(), case["group"]
    out = s["out"].double()
    for i, n in enumerate(s["length"].tolist()):
        a, b = off[i], off[i + 1]
        see = torch.zeros((b - a, n + b - a), dtype=torch.bool)
        for w in range(b - a):
            line, at = [w], w
            while at > 0 and 0 <= par[a + at] < at:
                at = par[a + at]
                line.append(at)
            if at == 0:
                see[w, :n] = True
                see[w, [n + j for j in line]] = True
        see = see.to(out.device)
        used = s["pages"][i, :(n + case["page"] - 1) // case["page"]].long()
        for h in range(case["kv_heads"]):
            k, v = (torch.cat([s[c + "_cache"][0, used, h].reshape(-1, case["dim"])[:n],
                               s[c][a:b, h]]).double() for c in "kv")
            for g in range(G):
                e = (s["q"][a:b, h * G + g].double() @ k.T) * s["scale"]
                e = torch.softmax(e.masked_fill(~see, -math.inf), 1).nan_to_num(0.0)
                out[a:b, h * G + g] = e @ v
    return {"out": out}


def _exact_verify(case, s):
    """Each window by itself, one node after the other, in numpy."""
    import numpy as np
    logits, tok, par, u = (s[k].cpu().numpy() for k in ("logits", "tokens", "parent", "u_accept"))
    off, temp, us = (s[k].cpu().numpy() for k in ("win_off", "temperature", "u_sample"))
    draft = s["draft_probs"].cpu().numpy() if case["sampled"] else None
    n, W, V = case["seqs"], case["window"], case["vocab"]
    path, nxt = -np.ones((n, W), np.int32), -np.ones(n, np.int32)
    n_path, prob = np.zeros(n, np.int32), np.zeros(logits.shape[0])
    for i in range(n):
        a, b = int(off[i]), int(off[i + 1])
        hangs = [True] + [False] * (b - a - 1)
        for w in range(1, b - a):
            hangs[w] = 0 <= par[a + w] < w and hangs[par[a + w]]
        prob[a], at = 1.0, 0
        for w in range(b - a):
            if not hangs[w]:
                continue
            x = logits[a + w].astype(np.float64)
            if temp[i] > 0:
                r = np.exp((x - x.max()) / np.float64(temp[i]))
                r /= r.sum()
            else:
                r = np.zeros(V)
                r[np.argmax(x)] = 1
            found = -1
            for c in range(w + 1, b - a):
                if not (hangs[c] and par[a + c] == w):
                    continue
                q = draft[a + c].astype(np.float64) if case["sampled"] else None
                qc = q[tok[a + c]] if case["sampled"] else 1.0
                rc = r[tok[a + c]]
                prob[a + c] = min(1.0, rc / qc) if qc > 0 else float(rc > 0)
                if found < 0 and u[a + c] * qc < rc:
                    found = c
                if case["sampled"]:
                    rest = np.maximum(r - q, 0)
                else:
                    rest = r.copy()
                    rest[tok[a + c]] = 0
                if rest.sum() >= REST:
                    r = rest / rest.sum()
            if w == at:
                path[i, n_path[i]] = w
                n_path[i] += 1
                if found >= 0:
                    at = found
                else:
                    cdf = np.cumsum(r)
                    nxt[i] = np.searchsorted(cdf, np.float64(us[i]) * cdf[-1], side="right")
    dev = s["logits"].device
    return {"path": torch.from_numpy(path).to(dev), "n_path": torch.from_numpy(n_path).to(dev),
            "next": torch.from_numpy(nxt).to(dev), "prob": torch.from_numpy(prob).to(dev)}


def _exact_commit(case, s):
    off, path, count = s["win_off"].tolist(), s["path"].tolist(), s["n_path"].tolist()
    length, pages = s["length"].tolist(), s["pages"].tolist()
    k, v = s["k_cache"].clone(), s["v_cache"].clone()
    for i in range(case["seqs"]):
        for j in range(count[i]):
            p = length[i] + j
            page, slot, row = pages[i][p // case["page"]], p % case["page"], off[i] + path[i][j]
            k[:, page, :, slot] = s["k"][:, row]
            v[:, page, :, slot] = s["v"][:, row]
    return {"k": k.double(), "v": v.double(),
            "length": _ints([x + c for x, c in zip(length, count)])}


def exact(case, seed):
    s = {"norm": _prepare_norm, "attn": _prepare_attn, "verify": _prepare_verify,
         "commit": _prepare_commit}[case["kind"]](case, seed)
    return {"norm": _exact_norm, "attn": _exact_attn, "verify": _exact_verify,
            "commit": _exact_commit}[case["kind"]](case, s)
