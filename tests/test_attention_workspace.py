"""A workspace that serves a call serves every smaller one: fewer sequences, shorter windows, shorter
caches (CPU: a call that gets its output over its windows is refused after its workspace is looked at,
and launches nothing)."""
import ctypes
import math
import random
import re

import pytest

import sager_amd

P = ctypes.c_void_p
INVALID, UNSUPPORTED = 1, 8
FAR = 1 << 44  # between buffers


@pytest.fixture(scope="module")
def lib():
    return sager_amd.load()


class Sliding:
    def __init__(self, lib, n_kv, group, D, reach, sinks):
        self.lib, self.heads, self.n_kv, self.D, self.more = lib, n_kv * group, n_kv, D, (reach, sinks)
        self.cache = sager_amd.KvCacheDesc(FAR, FAR * 2, FAR * 3, FAR * 4, 1 << 20, 1, 8, 16, 1 << 20,
                                           n_kv, D)
        self.entry, self.size = lib.sg_attn_sliding_f16, lib.sg_attn_sliding_workspace_bytes

    def bytes(self, n_seq, window, length):
        return self.size(n_seq, window, length, self.heads, self.n_kv, self.D, *self.more)

    def need(self, n_seq, window, length, given):
        """What the call needs beyond `given` bytes; None if they do, or if it is refused as it is."""
        kv = self.n_kv * self.D
        status = self.entry(P(FAR * 5), P(FAR * 6), P(FAR * 7), self.heads * self.D, kv, kv,
                            ctypes.byref(self.cache), 0, P(FAR * 8), None, P(FAR * 8), P(FAR * 9), given,
                            n_seq, 1, window, length, self.heads, 0.1, *self.more, None)
        if status == UNSUPPORTED:
            return None
        assert status == INVALID
        said = self.lib.sg_last_error().decode()
        if "overlaps the cache, win_off" in said:
            return None
        return int(re.search(r"needs (\d+) bytes", said)[1])


class Tree(Sliding):
    def __init__(self, lib, n_kv, group, D, *_):
        super().__init__(lib, n_kv, group, D, 0, 0)
        self.entry, self.size, self.more = lib.sg_attn_tree_f16, lib.sg_attn_tree_workspace_bytes, ()


def spread(rng, most):  # from 1 on, over the logarithm
    return round(2 ** rng.uniform(0, math.log2(most)))


def test_decoding_with_the_workspace_of_a_chunk(lib):
    c = Sliding(lib, 2, 8, 256, 0, 0)
    given = c.bytes(4, 4096, 32768)
    for window in (1, 4, 64, 1024, 4032):
        for length in (0, 1000, 32768):
            assert c.need(4, window, length, given) is None, (window, length)
    # and what is never cut needs none
    assert c.bytes(4, 1, 100) == 0


@pytest.mark.parametrize("seed", range(8))
def test_sliding(lib, seed):
    rng = random.Random(seed)
    for _ in range(1500):
        c = Sliding(lib, rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), rng.choice([1, 2, 3, 4, 5, 7, 8, 16, 40, 200]),
                    rng.choice([64, 128, 256]), rng.choice([0, spread(rng, 10000)]),
                    rng.choice([0, 4, 70, 5000]))
        most = spread(rng, 700), spread(rng, rng.choice([64, 8192])), spread(rng, 300000) - 1
        given = c.bytes(*most)
        for _ in range(12):
            less = spread(rng, most[0]), spread(rng, most[1]), spread(rng, most[2] + 1) - 1
            for call in (less, (less[0], most[1], less[2]), (most[0], less[1], most[2]),
                         (most[0], less[1], 0)):
                assert c.need(*call, given) is None, (c.__dict__, most, call)
                assert c.bytes(*call) <= given, (c.__dict__, most, call)


@pytest.mark.parametrize("seed", range(8))
def test_trees(lib, seed):
    rng = random.Random(100 + seed)
    for _ in range(1500):
        c = Tree(lib, rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), rng.choice([1, 2, 3, 4, 5, 7, 8, 16, 40]),
                 rng.choice([64, 128, 256]))
        most = spread(rng, 700), spread(rng, 64), spread(rng, 300000) - 1
        given = c.bytes(*most)
        for _ in range(12):
            less = spread(rng, most[0]), spread(rng, most[1]), spread(rng, most[2] + 1) - 1
            for call in (less, (most[0], less[1], most[2]), (most[0], most[1], less[2])):
                assert c.need(*call, given) is None, (c.__dict__, most, call)
                assert c.bytes(*call) <= given, (c.__dict__, most, call)


def test_sizes_past_all_calls(lib):
    most = 0x7FFFFFFF
    for heads, n_kv in ((1, 1), (1 << 20, 1 << 10), (most, most), (most, 1)):
        assert lib.sg_attn_sliding_workspace_bytes(most, most, most, heads, n_kv, 256, 0, 0) >= 0
    # as many sequences as a call takes
    f = lib.sg_attn_sliding_workspace_bytes
    assert f(most, 1, 10 ** 6, 2, 2, 64, 0, 0) == f(0x1FFFFF // 2, 1, 10 ** 6, 2, 2, 64, 0, 0) > 0
