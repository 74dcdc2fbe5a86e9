"""The operators around a quantised or a sliding cache, as cases that can be timed.

Between a layer's projections and its attention lie the heads' norms and the
rotary positions; the accepted tokens' keys and values then go into a cache.
A long context costs less if the cache holds 8 bits a value, or if a token
looks back over a window only, with the first few tokens (the sinks) in sight
throughout.  One kind of case for each:

  rope    the heads' RMS norms and rotary positions of q and k.
  store   keys and values quantised as they are written behind the cache (the
          accepted path of a verify window, or a prompt's whole chunk), then
          the sequences as they are read back.
  read    a range of a quantised cache's tokens as 16-bit rows.
  attn    a window's or a chunk's attention over a 16-bit or a quantised cache,
          over all of it or over a sliding window and the sinks.

Each case runs one operator: in its plain form, elementary torch operations
(`own` false), or by the library's entry point (`own` true).
"""
import math

import torch

own = False

DEVICE = "cuda"
GROUP = 32         # values of a quantised cache that share a scale
MOST_SCALE = 515.5  # 127 of these are still a 16-bit number


def listed():
    return [
        # a verify window of four behind 4,099 tokens: head norms, a quarter of the head rotated
        {"name": "rope_t4", "kind": "rope", "seqs": 1, "window": 4, "ragged": False, "branch": 1,
         "absent": False, "pad": 0, "len_lo": 4099, "len_hi": 4099, "heads": 16, "kv_heads": 2,
         "dim": 256, "rot": 64, "inter": False, "norm": True, "dtype": "f16", "scaling": "none",
         "given": False},
        # ragged trees of a padded batch far into a stretched context, neighbouring pairs
        {"name": "rope_trees_f32", "kind": "rope", "seqs": 9, "window": 13, "ragged": True,
         "branch": 3, "absent": True, "pad": 5, "len_lo": 0, "len_hi": 524287, "heads": 15,
         "kv_heads": 5, "dim": 64, "rot": 64, "inter": True, "norm": False, "dtype": "f32",
         "scaling": "yarn", "given": False},
        # a prompt's chunk at given positions, all of the head
        {"name": "rope_t4096", "kind": "rope", "seqs": 1, "window": 4096, "ragged": False,
         "branch": 1, "absent": False, "pad": 0, "len_lo": 126976, "len_hi": 126976, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "inter": False, "norm": True, "dtype": "f16",
         "scaling": "linear", "given": True},
        # the accepted part of a window of four, ten attention layers
        {"name": "store_t4_l10", "kind": "store", "seqs": 1, "window": 4, "ragged": False,
         "path": True, "layers": 10, "kv_heads": 2, "dim": 256, "len_lo": 59, "len_hi": 59,
         "page": 64},
        # prompts' ragged chunks behind what the sequences have
        {"name": "store_chunks", "kind": "store", "seqs": 5, "window": 1021, "ragged": True,
         "path": False, "layers": 10, "kv_heads": 8, "dim": 128, "len_lo": 0, "len_hi": 130,
         "page": 16},
        # a few tokens of one layer
        {"name": "read_t16", "kind": "read", "seqs": 1, "count": 16, "ragged": False, "layers": 1,
         "kv_heads": 2, "dim": 256, "first": 4090, "page": 64},
        # a conversation's cache, all attention layers, as it is kept between turns
        {"name": "read_32k_l10", "kind": "read", "seqs": 1, "count": 32749, "ragged": False,
         "layers": 10, "kv_heads": 2, "dim": 256, "first": 0, "page": 64},
        # a chain of four at the end of a long context of which a window is left
        {"name": "slide_chain4_128k", "kind": "attn", "cache": "f16", "reach": 4096, "sinks": 4,
         "evict": True, "seqs": 1, "window": 4, "ragged": False, "branch": 1, "absent": False,
         "pad": 0, "kv_heads": 2, "group": 8, "dim": 256, "len_lo": 131071, "len_hi": 131071,
         "page": 64},
        # sequences decoded together, one token each
        {"name": "slide_batch_q8", "kind": "attn", "cache": "q8", "reach": 1024, "sinks": 4,
         "evict": False, "seqs": 48, "window": 1, "ragged": False, "branch": 1, "absent": False,
         "pad": 0, "kv_heads": 8, "group": 4, "dim": 128, "len_lo": 77, "len_hi": 4001, "page": 16},
        # ragged trees over all of a quantised cache, a sequence without one
        {"name": "tree_batch_q8", "kind": "attn", "cache": "q8", "reach": 0, "sinks": 0,
         "evict": False, "seqs": 7, "window": 13, "ragged": True, "branch": 3, "absent": True,
         "pad": 5, "kv_heads": 5, "group": 3, "dim": 64, "len_lo": 0, "len_hi": 9001, "page": 32},
        # a chain of four over all of a long quantised context
        {"name": "chain4_128k_q8", "kind": "attn", "cache": "q8", "reach": 0, "sinks": 0,
         "evict": False, "seqs": 1, "window": 4, "ragged": False, "branch": 1, "absent": False,
         "pad": 0, "kv_heads": 2, "group": 8, "dim": 256, "len_lo": 131071, "len_hi": 131071,
         "page": 64},
        # a prompt's chunk behind 4,099 tokens, a sliding window: the largest
        {"name": "slide_chunk4096", "kind": "attn", "cache": "f16", "reach": 2048, "sinks": 4,
         "evict": False, "seqs": 1, "window": 4096, "ragged": False, "branch": 0, "absent": False,
         "pad": 0, "kv_heads": 2, "group": 8, "dim": 256, "len_lo": 4099, "len_hi": 4099,
         "page": 64},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "store", "store", "read", "attn", "attn", "attn", "attn"])
    seqs = _log_int(rng, 1, 32)
    if kind == "rope":
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        kv_heads = rng.randint(1, 8)
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        most = max(1, 4096 * 40 * 128 // (seqs * (heads + kv_heads) * dim))
        chunk = rng.random() < 0.5
        window = _log_int(rng, 1, min(4096 if chunk else 64, most))
        branch = 1 if chunk else rng.choice([1, 1, 2, 3, 5])
        lo = rng.choice([0, 13, _log_int(rng, 1, 131072)])
        return {"kind": kind, "seqs": seqs, "window": window,
                "ragged": seqs > 1 and rng.random() < 0.6, "branch": branch,
                "absent": branch > 1 and rng.random() < 0.4, "pad": rng.choice([0, 0, 1, 9]),
                "len_lo": lo, "len_hi": lo + _log_int(rng, 1, 500000), "heads": heads,
                "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)]),
                "inter": rng.random() < 0.5, "norm": rng.random() < 0.5,
                "dtype": rng.choice(["f16", "f16", "f32"]),
                "scaling": rng.choice(["none", "linear", "yarn"]), "given": window > 64}
    if kind == "store":
        kv_heads, dim, layers = rng.randint(1, 8), rng.choice([64, 128, 256]), _log_int(rng, 1, 40)
        path = rng.random() < 0.5
        lo = rng.choice([0, 13, _log_int(rng, 1, 500)])
        # tokens of a sequence, so that the largest listed case is not passed
        most = max(2, 3000 * 10 * 8 * 128 // (seqs * layers * kv_heads * dim))
        window = _log_int(rng, 1, min(64 if path else 4096, most))
        lo = min(lo, most)
        return {"kind": kind, "seqs": seqs, "window": window, "ragged": rng.random() < 0.5,
                "path": path, "layers": layers, "kv_heads": kv_heads, "dim": dim, "len_lo": lo,
                "len_hi": lo + _log_int(rng, 1, 100), "page": rng.choice([16, 32, 64])}
    if kind == "read":
        kv_heads, dim, layers = rng.randint(1, 8), rng.choice([64, 128, 256]), _log_int(rng, 1, 40)
        most = max(1, 32000 * 10 * 2 * 256 // (seqs * layers * kv_heads * dim))
        return {"kind": kind, "seqs": seqs, "count": _log_int(rng, 1, min(most, 40000)),
                "ragged": seqs > 1 and rng.random() < 0.5, "layers": layers, "kv_heads": kv_heads,
                "dim": dim, "first": rng.choice([0, 5, rng.randint(1, 1000)]),
                "page": rng.choice([16, 32, 64, 128])}
    dim = rng.choice([64, 128, 128, 256])
    kv_heads, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16])
    chunk = rng.random() < 0.4
    branch = 0 if chunk else rng.choice([1, 1, 2, 3, 5])
    # the largest listed case has 1.7e8 scores; a cache of 1.3e8 keys and values
    most = 1.3e8 / (2 * seqs * kv_heads * dim)
    rows = 1.7e8 / (seqs * kv_heads * group)
    window = _log_int(rng, 1, max(1, min(4096 if chunk else 64, most / 2, math.sqrt(rows / 2))))
    hi = _log_int(rng, 1, max(2, min(131072, most, rows / window)))
    reach = rng.choice([0, 1, _log_int(rng, 2, 8192), _log_int(rng, 2, 8192)])
    return {"kind": kind, "cache": rng.choice(["f16", "q8", "q8"]), "reach": reach,
            "sinks": 0 if reach == 0 else rng.choice([0, 1, 4, rng.randint(2, 300)]),
            "evict": reach > 0 and rng.random() < 0.5, "seqs": seqs, "window": window,
            "ragged": seqs > 1 and rng.random() < 0.6, "branch": branch,
            "absent": branch > 1 and rng.random() < 0.4, "pad": rng.choice([0, 0, 1, 9]),
            "kv_heads": kv_heads, "group": group, "dim": dim,
            "len_lo": rng.choice([0, hi, rng.randint(0, hi)]), "len_hi": hi,
            "page": rng.choice([16, 32, 64, 128])}


# ---- inputs -------------------------------------------------------------------

def _generator(seed, salt):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed * 1000003 + salt)
    return g


def _normal(gen, *shape, scale=1.0, dtype=torch.float16):
    return (torch.randn(shape, device=DEVICE, generator=gen) * scale).to(dtype)


def _sizes(most, n, ragged):
    """The windows' sizes: whole windows, or sizes from 1 up to the largest."""
    return [1 + (i * 7 + most - 1) % most for i in range(n)] if ragged else [most] * n


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


def _pages(gen, page, lengths, gone=None):
    """A table of pages in the pool's random order; entries past a sequence's last page are -1, and
    so are the pages that hold the tokens gone[i][0] .. gone[i][1] - 1 and nothing else."""
    per_seq = max(1, max((n + page - 1) // page for n in lengths))
    kept = []
    for i, n in enumerate(lengths):
        lo, hi = gone[i] if gone else (0, 0)
        first, last = (lo + page - 1) // page, hi // page
        kept.append([p for p in range((n + page - 1) // page) if not first <= p < last])
    n_pages = sum(len(k) for k in kept) + 3
    order = torch.randperm(n_pages, generator=gen, device=DEVICE).to(torch.int32)
    table, at = torch.full((len(lengths), per_seq), -1, dtype=torch.int32, device=DEVICE), 0
    for i, k in enumerate(kept):
        table[i, _ints(k, torch.int64)] = order[at:at + len(k)]
        at += len(k)
    return table, n_pages


BASE = 1e6          # of the rotary frequencies
FACTOR = 4.0        # contexts this many times longer than those trained on
TRAINED = 32768


def _frequencies(case):
    """Radians a position of each pair of the head's values, and what sine and cosine are
    multiplied by."""
    half = case["rot"] // 2
    i = torch.arange(half, dtype=torch.float64)
    f = BASE ** (-2 * i / case["rot"])
    if case["scaling"] == "linear":
        return f / FACTOR, 1.0
    if case["scaling"] == "yarn":
        # pairs that turn more than 32 times in a trained context stay, those that turn less than
        # once are stretched, with a ramp between them
        def pair(turns):
            return (case["rot"] * math.log(TRAINED / (turns * 2 * math.pi))
                    / (2 * math.log(BASE)))
        lo = max(math.floor(pair(32.0)), 0)
        hi = min(math.ceil(pair(1.0)), case["rot"] - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / FACTOR * ramp + f * (1 - ramp), 0.1 * math.log(FACTOR) + 1
    return f, 1.0


def _prepare_rope(case, seed):
    gen = _generator(seed, 1)
    dt = torch.float16 if case["dtype"] == "f16" else torch.float32
    sizes, lengths = _sizes(case["window"], case["seqs"], case["ragged"]), _lengths(case)
    off = _offsets(sizes)
    T, H, K, D = off[-1] + case["pad"], case["heads"], case["kv_heads"], case["dim"]
    # q, k and v are slices of one projection's output
    qkv = _normal(gen, T, (H + 2 * K) * D, scale=1.5, dtype=dt)
    q, k, _ = qkv.split([H * D, K * D, K * D], dim=1)
    freq, mscale = _frequencies(case)
    state = {"q": q.view(T, H, D), "k": k.view(T, K, D), "freq": freq.to(DEVICE),
             "mscale": mscale, "eps": 1e-6, "win_off": _ints(off), "length": _ints(lengths),
             "parent": None if case["given"] else _ints(_parents(case, sizes)),
             "positions": None, "q_norm": None, "k_norm": None,
             "q_out": torch.zeros((T, H, D), dtype=dt, device=DEVICE),
             "k_out": torch.zeros((T, K, D), dtype=dt, device=DEVICE)}
    if case["given"]:
        state["positions"] = torch.cat(
            [_ints(list(range(n, n + s))) for n, s in zip(lengths, sizes)]
            + [torch.zeros(case["pad"], dtype=torch.int32, device=DEVICE)])
    if case["norm"]:
        for name in ("q_norm", "k_norm"):
            state[name] = 1 + 0.2 * torch.randn(D, device=DEVICE, generator=gen)
    return state


def _quantise(x):
    """8-bit codes and 16-bit scales of groups of 32 values."""
    g = x.float().unflatten(-1, (-1, GROUP))
    scale = (g.abs().amax(-1, keepdim=True) / 127).half().float().clamp_max(MOST_SCALE)
    code = (g / torch.where(scale > 0, scale, 1)).round().clamp(-127, 127)
    return code.flatten(-2).to(torch.int8), scale[..., 0].half()


def _values(code, scale):
    return (code.float().unflatten(-1, (-1, GROUP)) * scale.float()[..., None]).flatten(-2)


def _pool(case, gen, layers, n_pages, q8):
    """Keys' and values' pages, some channels of the keys larger than the others."""
    pool = {}
    for name in ("k", "v"):
        x = _normal(gen, layers, n_pages, case["kv_heads"], case["page"], case["dim"])
        if name == "k":
            x[..., 3::41] *= 3
        if q8:
            pool[name + "_cache"], pool[name + "_scale"] = _quantise(x)
        else:
            pool[name + "_cache"] = x
    return pool


def _prepare_store(case, seed):
    gen = _generator(seed, 2)
    sizes, lengths = _sizes(case["window"], case["seqs"], case["ragged"]), _lengths(case)
    off, n, W = _offsets(sizes), case["seqs"], case["window"]
    L, T, H, D = case["layers"], off[-1], case["kv_heads"], case["dim"]
    pages, n_pages = _pages(gen, case["page"], [a + b for a, b in zip(lengths, sizes)])
    state = {"k": _normal(gen, L, T, H, D), "v": _normal(gen, L, T, H, D), "pages": pages,
             "length": _ints(lengths), "win_off": _ints(off), "path": None, "n_path": None,
             # what is read back: every sequence from its first token, as if all were accepted
             "first": _ints([0] * n),
             "rows": _ints(_offsets([a + b for a, b in zip(lengths, sizes)]))}
    state.update(_pool(case, gen, L, n_pages, True))
    if case["path"]:
        # accepted paths as a verification leaves them: the root and some descendants, in order
        size, node = _ints(sizes, torch.int64), torch.arange(W, device=DEVICE)
        keep = torch.rand((n, W), device=DEVICE, generator=gen) < 0.7
        keep = (keep | (node == 0)) & (node < size[:, None])
        path = torch.where(keep, node, W).sort(1).values
        state["path"] = torch.where(path < W, path, -1).to(torch.int32)
        state["n_path"] = keep.sum(1).to(torch.int32)
    return state


def _prepare_read(case, seed):
    gen = _generator(seed, 3)
    sizes = _sizes(case["count"], case["seqs"], case["ragged"])
    lengths = [case["first"] + s for s in sizes]
    pages, n_pages = _pages(gen, case["page"], lengths)
    return {"pages": pages, "length": _ints(lengths), "first": _ints([case["first"]] * len(sizes)),
            "rows": _ints(_offsets(sizes)), **_pool(case, gen, case["layers"], n_pages, True)}


def _prepare_attn(case, seed):
    gen = _generator(seed, 4)
    sizes, lengths = _sizes(case["window"], case["seqs"], case["ragged"]), _lengths(case)
    off = _offsets(sizes)
    T, H, G, D = off[-1] + case["pad"], case["kv_heads"], case["group"], case["dim"]
    # what no token of a window sees any more, if its pages have gone to others
    gone = [(case["sinks"], max(0, n - case["reach"] + 1)) for n in lengths]
    pages, n_pages = _pages(gen, case["page"], lengths, gone if case["evict"] else None)
    # q, k and v of the window are slices of one projection's output
    qkv = _normal(gen, T, (H * G + 2 * H) * D)
    q, k, v = qkv.split([H * G * D, H * D, H * D], dim=1)
    q.mul_(2.0)
    return {"q": q.view(T, H * G, D), "k": k.view(T, H, D), "v": v.view(T, H, D),
            "pages": pages, "length": _ints(lengths), "win_off": _ints(off),
            "parent": _ints(_parents(case, sizes)) if case["branch"] else None,
            "scale": 1 / math.sqrt(D),
            "out": torch.zeros((T, H * G, D), dtype=torch.float16, device=DEVICE),
            **_pool(case, gen, 1, n_pages, case["cache"] == "q8")}


_PREPARE = {"rope": _prepare_rope, "store": _prepare_store, "read": _prepare_read,
            "attn": _prepare_attn}


def prepare(case, seed):
    state = _PREPARE[case["kind"]](case, seed)
    state["case"] = case
    if own:
        _handles(case, state)
    return state


def _handles(case, state):
    """What a program keeps for the library's calls: tables, caches, objects with workspaces, and
    output buffers."""
    from sager_amd import ops
    if case["kind"] == "rope":
        scaling = {"none": {}, "linear": {"scaling": "linear", "factor": FACTOR},
                   "yarn": {"scaling": "yarn", "factor": FACTOR, "trained": TRAINED}}
        state["table"] = ops.rope_frequencies(case["rot"], BASE, **scaling[case["scaling"]])
        return
    if "k_scale" in state:
        state["cache"] = ops.KvCacheQ8(state["k_cache"], state["v_cache"], state["k_scale"],
                                       state["v_scale"], state["pages"], state["length"])
    else:
        state["cache"] = ops.KvCache(state["k_cache"], state["v_cache"], state["pages"],
                                     state["length"])
    if case["kind"] == "attn":
        state["attn"] = ops.SlidingAttention(
            case["kv_heads"] * case["group"], case["kv_heads"], case["dim"],
            max_tokens=state["q"].shape[0], max_seqs=case["seqs"], max_window=case["window"],
            max_len=case["len_hi"], reach=case["reach"], sinks=case["sinks"])
    else:
        n = state["k"].shape[1] + sum(_lengths(case)) if case["kind"] == "store" else \
            sum(_sizes(case["count"], case["seqs"], case["ragged"]))
        shape = (case["layers"], n, case["kv_heads"], case["dim"])
        state["k_out"], state["v_out"] = (torch.empty(shape, dtype=torch.float16, device=DEVICE)
                                          for _ in range(2))


# ---- the plain forms ------------------------------------------------------------

def _rows(off, window):
    """Rows of the windows' nodes [n, window], and which of them there are."""
    off = off.long()
    node = torch.arange(window, device=off.device)
    row = off[:-1, None] + node
    there = row < off[1:, None]
    return torch.where(there, row, 0), there


def _tree(state, window):
    """Rows of the windows' nodes [n, W], which of them there are, and who is whose ancestor
    (or the node itself) [n, W, W]; a node that does not hang on its window's first is absent."""
    row, there = _rows(state["win_off"], window)
    node = torch.arange(window, device=row.device)
    if state["parent"] is None:
        return row, there, (node[:, None] >= node) & there[:, :, None]
    par = torch.where(there, state["parent"].long()[row], -1)
    edge = (par >= 0) & (par < node) & (node > 0)
    up = (node[:, None] == node) | (edge[:, :, None] & (par[:, :, None] == node))
    up = up.float()
    for _ in range(max(1, (window - 1).bit_length())):
        up = (up @ up).clamp_max(1)
    there = there & (up[:, :, 0] > 0)
    return row, there, (up > 0) & there[:, :, None]


def _plain_rope(state):
    case = state["case"]
    if case["given"]:
        rows = torch.arange(state["q"].shape[0], device=DEVICE)
        pos = state["positions"].double()
    else:
        row, there, up = _tree(state, case["window"])
        rows = row[there]
        pos = (state["length"].long()[:, None] + up.sum(2) - 1)[there].double()
    angle = pos[:, None] * state["freq"]
    cos, sin = ((f(angle) * state["mscale"]).float()[:, None] for f in (torch.cos, torch.sin))
    got, r = {}, case["rot"]
    for name in ("q", "k"):
        x = state[name][rows].float()
        if case["norm"]:
            x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + state["eps"]) \
                * state[name + "_norm"]
        a, b = (slice(0, r, 2), slice(1, r, 2)) if case["inter"] else \
            (slice(0, r // 2), slice(r // 2, r))
        y = x.clone()
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
        out = state[name + "_out"]
        out[rows] = y.to(out.dtype)
        got[name] = out
    return got


def _gather(state, rows, first, n):
    """Tokens first[s] + i of each sequence as rows rows[s] + i, n rows in all."""
    at = torch.arange(n, device=DEVICE)
    seq = torch.searchsorted(rows.long()[1:], at, right=True)
    pos = first.long()[seq] + at - rows.long()[seq]
    page = state["case"]["page"]
    at = state["pages"].long()[seq, pos // page]
    head = torch.arange(state["case"]["kv_heads"], device=DEVICE)

    def pick(c):
        return c[:, at[:, None], head, (pos % page)[:, None]]

    return {c: _values(pick(state[c + "_cache"]), pick(state[c + "_scale"])).half() for c in "kv"}


def _plain_store(state):
    case = state["case"]
    page, W = case["page"], case["window"]
    node = torch.arange(W, device=DEVICE)
    if case["path"]:
        count = state["n_path"].long()
        keep = node < count[:, None]
        row = (state["win_off"].long()[:-1, None] + state["path"].long())[keep]
    else:
        row, keep = _rows(state["win_off"], W)
        count, row = keep.sum(1), row[keep]
    pos = state["length"].long()[:, None] + node
    pos = torch.where(keep, pos, 0)
    at, pos = state["pages"].long().gather(1, pos // page)[keep], pos[keep]
    head = torch.arange(case["kv_heads"], device=DEVICE)
    for name in ("k", "v"):
        code, scale = _quantise(state[name][:, row])
        state[name + "_cache"][:, at[:, None], head, (pos % page)[:, None]] = code
        state[name + "_scale"][:, at[:, None], head, (pos % page)[:, None]] = scale
    n = state["k"].shape[1] + sum(_lengths(case))
    return {**_gather(state, state["rows"], state["first"], n),
            "length": (state["length"] + count).to(torch.int32)}


def _plain_read(state):
    case = state["case"]
    n = sum(_sizes(case["count"], case["seqs"], case["ragged"]))
    return _gather(state, state["rows"], state["first"], n)


def _plain_attn(state):
    case = state["case"]
    n, W, H, G, D = (case[c] for c in ("seqs", "window", "kv_heads", "group", "dim"))
    row, there, up = _tree(state, W)
    length = state["length"].long()[:, None]
    at = length + up.sum(2) - 1  # the nodes' positions
    sinks, reach = case["sinks"], case["reach"]
    # the cached tokens that anyone sees: the sinks, and what the first node looks back on
    if reach == 0 or sinks + reach > case["len_hi"]:
        pos = torch.arange(case["len_hi"], device=DEVICE).expand(n, -1)
        seen = pos < length
    else:
        low = (length - reach + 1).clamp_min(0)
        low = torch.maximum(low, torch.full_like(low, sinks))
        pos = torch.cat([torch.arange(sinks, device=DEVICE).expand(n, -1),
                         low + torch.arange(reach - 1, device=DEVICE)], 1)
        seen = pos < length
    pos = torch.where(seen, pos, 0)
    if pos.shape[1]:
        slot = state["pages"].long().gather(1, pos // case["page"])
        seen = seen & (slot >= 0)
        slot = slot.clamp_min(0)
    else:
        slot = pos
    head = torch.arange(H, device=DEVICE)

    def cached(c):  # [n, H, len, D]
        i = (slot[:, None, :], head[None, :, None], (pos % case["page"])[:, None, :])
        if case["cache"] == "q8":
            return _values(state[c + "_cache"][0][i], state[c + "_scale"][0][i])
        return state[c + "_cache"][0][i].float()

    q = state["q"][row].float().view(n, W, H, G, D).permute(0, 2, 1, 3, 4).reshape(n, H, W * G, D)
    k_new = state["k"][row].float().transpose(1, 2).contiguous()
    v_new = state["v"][row].float().transpose(1, 2).contiguous()
    k = torch.cat([cached("k"), k_new], 2)
    s = q @ k.transpose(2, 3).contiguous() * state["scale"]
    mask = torch.cat([seen[:, None, :].expand(n, W, -1), up], 2)
    if reach:
        key = torch.cat([pos, at], 1)[:, None, :]
        mask = mask & ((key < sinks) | (key > at[:, :, None] - reach))
    mask = (mask & there[:, :, None]).repeat_interleave(G, 1)[:, None]
    s = s.masked_fill_(~mask, -math.inf)
    top = s.amax(3, keepdim=True)
    e = torch.exp(s.sub_(torch.where(top > -math.inf, top, 0)))
    v = torch.cat([cached("v"), v_new], 2)
    total = e.sum(3, keepdim=True)
    o = e @ v / torch.where(total > 0, total, 1)
    o = o.view(n, H, W, G, D).permute(0, 2, 1, 3, 4).reshape(n, W, H * G, D).half()
    # (past a window's end, its first row once more)
    node = torch.arange(W, device=row.device)
    off = state["win_off"].long()
    node = torch.where(node < (off[1:] - off[:-1])[:, None], node, 0)
    state["out"][off[:-1, None] + node] = o[torch.arange(n, device=row.device)[:, None], node]
    return {"out": state["out"]}


# ---- the library's calls --------------------------------------------------------

def _own(state):
    from sager_amd import ops
    case = state["case"]
    if case["kind"] == "rope":
        where = {"positions": state["positions"]} if case["given"] else \
            {"win_off": state["win_off"], "parent": state["parent"], "length": state["length"]}
        q, k = ops.rope(state["q"], state["k"], state["table"], **where,
                        interleaved=case["inter"], mscale=state["mscale"],
                        q_norm=state["q_norm"], k_norm=state["k_norm"], eps=state["eps"],
                        q_out=state["q_out"], k_out=state["k_out"])
        return {"q": q, "k": k}
    if case["kind"] == "attn":
        return {"out": state["attn"].forward(
            state["q"], state["k"], state["v"], state["cache"], state["win_off"],
            state["parent"], scale=state["scale"], out=state["out"])}
    got = {}
    if case["kind"] == "store" and case["path"]:
        got["length"] = state["cache"].commit(state["k"], state["v"], state["win_off"],
                                              state["path"], state["n_path"])
    elif case["kind"] == "store":
        got["length"] = state["cache"].append(state["k"], state["v"], state["win_off"],
                                              case["window"])
    got["k"], got["v"] = state["cache"].read(state["first"], state["rows"], k_out=state["k_out"],
                                             v_out=state["v_out"])
    return got


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "store": _plain_store, "read": _plain_read,
            "attn": _plain_attn}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------

def _pairs(n, s, reach, sinks):
    """Keys that a chain of s tokens behind n cached ones sees, over all of its tokens."""
    return sum(p + 1 if reach == 0 else min(p + 1, reach + min(sinks, max(0, p + 1 - reach)))
               for p in range(n, n + s))


def work(case):
    kind = case["kind"]
    if kind == "read":
        rows = sum(_sizes(case["count"], case["seqs"], case["ragged"]))
        n = case["layers"] * rows * case["kv_heads"] * case["dim"]
        return {"bytes": 2.0 * n * (1 + 2 / GROUP + 2), "flops": 2.0 * n}
    sizes, lengths = _sizes(case["window"], case["seqs"], case["ragged"]), _lengths(case)
    if kind == "rope":
        n = sum(sizes) * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": (4.0 if case["dtype"] == "f16" else 8.0) * n, "flops": 8.0 * n}
    if kind == "store":
        one = 2.0 * case["layers"] * case["kv_heads"] * case["dim"]
        new = sum(1 + 0.7 * (s - 1) for s in sizes) if case["path"] else sum(sizes)
        return {"bytes": one * (new * (3 + 2 / GROUP)
                                + (sum(sizes) + sum(lengths)) * (3 + 2 / GROUP)),
                "flops": 4.0 * one * new}
    H, G, D, reach, sinks = (case[c] for c in ("kv_heads", "group", "dim", "reach", "sinks"))
    width = 2.0 if case["cache"] == "f16" else 1 + 2 / GROUP
    total = flops = 0
    for s, n in zip(sizes, lengths):
        seen = n if reach == 0 else min(n, reach - 1 + min(sinks, max(0, n - reach + 1)))
        total += 2 * width * seen * H * D + 4.0 * s * H * D + 4.0 * s * H * G * D
        flops += 4.0 * H * G * D * _pairs(n, s, reach, sinks)
    return {"bytes": total, "flops": flops}


# ---- the same in 64 bits ----------------------------------------------------------

def _line(par, a, w):
    """Node w of the window at row a and its ancestors; empty if it does not hang on the first."""
    line = [w]
    while w > 0:
        up = w - 1 if par is None else par[a + w]
        if not 0 <= up < w:
            return []
        line.append(up)
        w = up
    return line


def _exact_rope(case, s):
    off, length = s["win_off"].tolist(), s["length"].tolist()
    par = None if s["parent"] is None else s["parent"].tolist()
    pos = [None] * s["q"].shape[0]
    if case["given"]:
        pos = s["positions"].tolist()
    else:
        for i, n in enumerate(length):
            for w in range(off[i + 1] - off[i]):
                line = _line(par, off[i], w)
                pos[off[i] + w] = n + len(line) - 1 if line else None
    rows = [t for t, p in enumerate(pos) if p is not None]
    p = _ints([pos[t] for t in rows], torch.float64)
    turn = torch.polar(torch.full((len(rows), case["rot"] // 2), s["mscale"], dtype=torch.float64,
                                  device=DEVICE), torch.outer(p, s["freq"]))[:, None]
    got, rows = {}, _ints(rows, torch.int64)
    for name in ("q", "k"):
        x = s[name][rows].double()
        if case["norm"]:
            x = x / (x.pow(2).sum(2, keepdim=True) / case["dim"] + s["eps"]).sqrt() \
                * s[name + "_norm"].double()
        head, tail = x[..., :case["rot"]], x[..., case["rot"]:]
        pair = head.unflatten(-1, (-1, 2)) if case["inter"] else \
            head.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z if case["inter"] else z.transpose(-1, -2)
        out = torch.zeros(s[name].shape, dtype=torch.float64, device=DEVICE)
        out[rows] = torch.cat([z.flatten(-2), tail], -1)
        got[name] = out
    return got


def _exact_tokens(s, name, i, lo, hi, page):
    """Tokens lo .. hi - 1 of sequence i: [layers, tokens, heads, dim]."""
    p = torch.arange(lo, hi, device=DEVICE)
    at = s["pages"][i].long()[p // page]
    c, d = (s[name + x].permute(1, 3, 0, 2, 4)[at, p % page] for x in ("_cache", "_scale"))
    return (c.double() * d.double().repeat_interleave(GROUP, -1)).transpose(0, 1)


def _exact_read(case, s):
    got = {}
    rows = s["rows"].tolist()
    for name in ("k", "v"):
        got[name] = torch.cat([
            _exact_tokens(s, name, i, case["first"], case["first"] + rows[i + 1] - rows[i],
                          case["page"]) for i in range(case["seqs"])], 1)
    return got


def _exact_store(case, s):
    """Sequence after sequence: the old tokens, then each new one by itself."""
    off, length, rows = s["win_off"].tolist(), s["length"].tolist(), s["rows"].tolist()
    new_length = []
    got = {"k": [], "v": []}
    for i, n in enumerate(length):
        size = off[i + 1] - off[i]
        nodes = s["path"][i, :int(s["n_path"][i])].tolist() if case["path"] else list(range(size))
        new_length.append(n + len(nodes))
        for name in ("k", "v"):
            seq = _exact_tokens(s, name, i, 0, rows[i + 1] - rows[i], case["page"])
            x = s[name][:, _ints([off[i] + w for w in nodes], torch.int64)].double()
            g = x.reshape(*x.shape[:-1], case["dim"] // GROUP, GROUP)
            step = (g.abs().max(-1)[0] / 127).to(torch.float16).double()
            step = step.clamp(max=MOST_SCALE)[..., None]
            y = torch.where(step > 0, torch.round(g / step).clamp(-127, 127) * step, 0)
            seq[:, n:n + len(nodes)] = y.reshape(x.shape)
            got[name].append(seq)
    return {"k": torch.cat(got["k"], 1), "v": torch.cat(got["v"], 1), "length": _ints(new_length)}


def _exact_attn(case, s):
    """One sequence and one head after the other."""
    off, G = s["win_off"].tolist(), case["group"]
    par = None if s["parent"] is None else s["parent"].tolist()
    out = s["out"].double()
    page, reach, sinks = case["page"], case["reach"] or 1 << 40, case["sinks"]
    for i, n in enumerate(s["length"].tolist()):
        a, b = off[i], off[i + 1]
        pos = torch.arange(n, device=DEVICE)
        pos = pos[(pos < sinks) | (pos > n - reach)]
        at = s["pages"][i].long()[pos // page] if len(pos) else pos
        pos, at = pos[at >= 0], at[at >= 0]
        w = b - a
        tree = torch.zeros((w, w), dtype=torch.bool)
        if par is None:
            tree = torch.ones((w, w), dtype=torch.bool).tril()
        else:
            for t in range(w):
                tree[t, _line(par, a, t)] = True
        tree = tree.to(DEVICE)
        mine = n + tree.sum(1) - 1
        key = torch.cat([pos, mine])
        see = torch.cat([tree.any(1)[:, None].expand(w, len(pos)), tree], 1)
        see = see & ((key < sinks) | (key > mine[:, None] - reach))
        for h in range(case["kv_heads"]):
            kv = []
            for c in "kv":
                x = s[c + "_cache"][0, at, h, pos % page].double()
                if case["cache"] == "q8":
                    x = x * s[c + "_scale"][0, at, h, pos % page].double() \
                        .repeat_interleave(GROUP, -1)
                kv.append(torch.cat([x, s[c][a:b, h].double()]))
            for g in range(G):
                e = (s["q"][a:b, h * G + g].double() @ kv[0].T) * s["scale"]
                e = torch.softmax(e.masked_fill_(~see, -math.inf), 1).nan_to_num_(0.0)
                out[a:b, h * G + g] = e @ kv[1]
    return {"out": out}


def exact(case, seed):
    s = _PREPARE[case["kind"]](case, seed)
    return {"rope": _exact_rope, "store": _exact_store, "read": _exact_read,
            "attn": _exact_attn}[case["kind"]](case, s)
