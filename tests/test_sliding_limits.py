"""Which batches the sliding attention takes: the limits are those of the launches that it makes (CPU:
a call that gets its output over its windows is refused behind them, and launches nothing)."""
import ctypes

import pytest

import sager_amd

P = ctypes.c_void_p
INVALID, UNSUPPORTED = 1, 8
FAR = 1 << 44  # between buffers


def call(n_seq, window, heads, n_kv, D, max_len=4096, reach=0, sinks=0, n_tokens=4):
    lib = sager_amd.load()
    c = sager_amd.KvCacheDesc(FAR, FAR * 2, FAR * 3, FAR * 4, 1 << 20, 1, 8, 16, 1 << 20, n_kv, D)
    status = lib.sg_attn_sliding_f16(P(FAR * 5), P(FAR * 6), P(FAR * 7), heads * D, n_kv * D, n_kv * D,
                                     ctypes.byref(c), 0, P(FAR * 8), None, P(FAR * 8), P(FAR * 9), 1 << 43,
                                     n_seq, n_tokens, window, max_len, heads, 0.1, reach, sinks, None)
    assert status == UNSUPPORTED or b"overlaps the cache, win_off" in lib.sg_last_error()
    return status == INVALID


@pytest.mark.parametrize("reach", [0, 1000])
def test_a_chunk_among_single_tokens(reach):
    """Bounds of a mixed batch: one sequence's chunk, the others' single tokens.  Nothing is cut, so
    nothing is joined, and the attention's own launch has room."""
    for n_seq, window, heads, n_kv, D in ((128, 2048, 64, 8, 128), (128, 4096, 32, 8, 128),
                                          (64, 8192, 32, 8, 128), (128, 4096, 64, 8, 64),
                                          (64, 8192, 16, 2, 256), (256, 4096, 32, 8, 128)):
        assert call(n_seq, window, heads, n_kv, D, reach=reach), (n_seq, window)


def test_launches_past_their_limits():
    # 2^23 workgroups of 256 rows, 2^21 units
    assert call((1 << 13) - 1, 1 << 13, 32, 8, 128) and not call(1 << 13, 1 << 13, 32, 8, 128)
    assert call((1 << 21) - 1, 1, 1, 1, 64, max_len=0) and not call(1 << 20, 1, 2, 2, 64, max_len=0)
    assert not call(1 << 30, 1, 1 << 30, 1 << 30, 256) and not call(0x7FFFFFFF, 1 << 24, 64, 64, 64)
    assert not call(1, 1 << 24, 256, 1, 64)
    # joins of 2^23 rows, of 512 threads each
    for max_len, cut in ((100000, True), (0, False)):
        assert call((1 << 16) - 1, 1, 128, 1, 256, max_len=max_len)
        assert call(1 << 16, 1, 128, 1, 256, max_len=max_len) != cut
