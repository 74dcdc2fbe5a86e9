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
