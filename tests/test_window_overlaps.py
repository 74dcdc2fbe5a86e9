"""Buffers of the verify window's entry points that share memory where one is written while others
are read: refused before any launch (no GPU)."""
import ctypes

import pytest

import sager_amd

P = ctypes.c_void_p
INVALID = 1
ROOM = 1 << 30  # between buffers


@pytest.fixture(scope="module")
def lib():
    return sager_amd.load()


def apart(*names):
    """Addresses far from each other, by name."""
    return {n: ROOM * (i + 1) for i, n in enumerate(names)}


def refused(call, what, lib):
    assert call() == INVALID, what
    assert b"overlap" in lib.sg_last_error(), (what, lib.sg_last_error())


def test_commit_lengths_over_what_is_read(lib):
    """n_path, path, win_off, the page table: read by workgroups that run beside the one that writes
    length_out."""
    a = apart("k", "v", "kc", "vc", "pages", "length", "off", "path", "n_path")
    c = sager_amd.KvCacheDesc(a["kc"], a["vc"], a["pages"], a["length"], 1 << 20, 2, 8, 16, 4, 2, 128)
    n_seq, W = 3, 4
    for name, ints in (("n_path", n_seq), ("path", n_seq * W), ("off", n_seq + 1),
                       ("pages", n_seq * 4), ("length", n_seq)):
        for at in (a[name], a[name] + 4 * (ints - 1), a[name] - 4 * (n_seq - 1)):
            args = [P(a["k"]), P(a["v"]), 256, 256, 4096, 4096, ctypes.byref(c), P(a["off"]),
                    P(a["path"]), P(a["n_path"]), P(at), n_seq, 4, W, None]
            refused(lambda: lib.sg_kv_commit_f16(*args), (name, at), lib)


@pytest.mark.parametrize("f16", [False, True])
def test_norm_outputs_over_other_rows(lib, f16):
    """x_out and xn may be x or y; shifted against them they are other rows' inputs, and in one place
    they are not two outputs."""
    fn, size = (lib.sg_add_rmsnorm_q8_k_f16, 2) if f16 else (lib.sg_add_rmsnorm_q8_k, 4)
    n, rows = 512, 5
    row, q8 = n * size, 2 * 276
    a = apart("x", "y", "x_out", "w", "xn", "xq")
    end = {"x": rows * row, "y": rows * row, "x_out": rows * row, "w": n * 4, "xn": rows * row,
           "xq": rows * q8}

    def call(**kw):
        b = dict(a, **kw)
        return fn(P(b["x"]), P(b["y"]), P(b["x_out"]), P(b["w"]), 1e-6, P(b["xn"]), P(b["xq"]), n,
                  rows, None)
    for out in ("x_out", "xn", "xq"):
        for other in set(a) - {out}:
            places = [a[other] + end[other] - 4, a[other] - end[out] + 4, a[other] + row]
            if out == "xq" or other in ("w", "xq") or {out, other} == {"x_out", "xn"}:
                places.append(a[other])
            for at in places:
                if a[other] - end[out] < at < a[other] + end[other]:
                    refused(lambda: call(**{out: at}), (out, other, at), lib)
    # both in x's place, and without the addition xq in x's
    refused(lambda: call(x_out=a["x"], xn=a["x"]), "one place", lib)
    assert fn(P(a["x"]), None, None, P(a["w"]), 1e-6, None, P(a["x"]), n, rows, None) == INVALID
    assert b"overlap" in lib.sg_last_error()


def test_verify_outputs_over_what_is_read(lib):
    n_seq, T, W, V = 3, 7, 4, 5000
    need = lib.sg_tree_verify_workspace_bytes(T, V, 2)
    size = dict(logits=T * V * 4, tokens=T * 4, off=(n_seq + 1) * 4, parent=T * 4, draft=T * V * 4,
                temp=n_seq * 4, ua=T * 4, us=n_seq * 4, path=n_seq * W * 4, n_path=n_seq * 4,
                next=n_seq * 4, prob=T * 4, ws=need)
    a = apart(*size)

    def call(**kw):
        b = [P(v) for v in dict(a, **kw).values()]
        return lib.sg_tree_verify(*b, need, n_seq, T, W, V, 2, None)
    for out in ("path", "n_path", "next", "prob"):
        for other in set(size) - {out}:
            for at in (a[other], a[other] + size[other] - 4, a[other] - size[out] + 4):
                refused(lambda: call(**{out: at}), (out, other, at), lib)


def test_attention_output_over_cache_and_workspace(lib):
    n_seq, T, W, heads, kv, D, n_pages, page, per = 3, 7, 4, 8, 2, 128, 9, 16, 4
    need = lib.sg_attn_tree_workspace_bytes(n_seq, W, 4000, heads, kv, D)
    assert need > 0
    layer = n_pages * kv * page * D
    size = dict(q=T * heads * D * 2, k=T * kv * D * 2, v=T * kv * D * 2, kc=layer * 2, vc=layer * 2,
                pages=n_seq * per * 4, length=n_seq * 4, off=(n_seq + 1) * 4, parent=T * 4, ws=need)
    a, n_out = apart(*size), T * heads * D * 2
    c = sager_amd.KvCacheDesc(a["kc"] - 2 * layer, a["vc"] - 2 * layer, a["pages"], a["length"],
                              layer, 2, n_pages, page, per, kv, D)
    for other in size:
        for at in (a[other], a[other] + (size[other] - 2) // 8 * 8, a[other] - n_out + 8):
            refused(lambda: lib.sg_attn_tree_f16(
                P(a["q"]), P(a["k"]), P(a["v"]), heads * D, kv * D, kv * D, ctypes.byref(c), 1,
                P(a["off"]), P(a["parent"]), P(at), P(a["ws"]), need, n_seq, T, W, 4000, heads, 0.1,
                None), (other, at), lib)
