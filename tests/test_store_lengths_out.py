"""New lengths over what a store still reads or writes are refused, in both caches, by path or of whole windows
(CPU: the calls are refused before anything is launched)."""
import ctypes

import pytest

import sager_amd

P = ctypes.c_void_p
INVALID = 1
ROOM = 1 << 30  # between buffers
N_SEQ, T, N_KV, D, PAGE, N_PAGES, LAYERS = 3, 4, 2, 128, 16, 8, 3
ROW, LD, LAYER_LD = N_KV * D, 700, 4096        # values of a token's k, from token to token, layer to layer
LAYER, LAYER_AT = N_PAGES * N_KV * PAGE * D, 1 << 17  # values of a layer, from layer to layer


@pytest.fixture(params=["f16", "q8"])
def q8(request):
    return request.param == "q8"


@pytest.fixture(params=["commit", "append"])
def store(request, q8):
    """store(where length_out is): is refused for that."""
    lib = sager_amd.load()
    fn = getattr(lib, f"sg_kv_{request.param}_{'q8' if q8 else 'f16'}")
    geo = (LAYER_AT, LAYERS, N_PAGES, PAGE, 4, N_KV, D)
    at = [P(ROOM * i) for i in range(20)]
    c = sager_amd.KvCacheQ8Desc(ROOM, ROOM * 2, ROOM * 3, ROOM * 4, ROOM * 5, ROOM * 6, *geo) if q8 else \
        sager_amd.KvCacheDesc(ROOM, ROOM * 2, ROOM * 5, ROOM * 6, *geo)
    path = [at[13], at[14]] if request.param == "commit" else []

    def call(out):
        status = fn(at[10], at[11], LD, LD, LAYER_LD, LAYER_LD, ctypes.byref(c), at[12], *path, P(out),
                    N_SEQ, T, 4, None)
        assert status == INVALID and b"length_out" in lib.sg_last_error(), (out, status)
    return call


@pytest.mark.parametrize("base", [10, 11])
def test_over_what_is_read(store, base):
    for layer in range(LAYERS):
        for t in range(T):
            row = ROOM * base + 2 * (layer * LAYER_LD + t * LD)
            for spot in (row, row + 2 * ROW - 4, row - 4 * N_SEQ + 4, row + ROW):
                store(spot)


def test_over_what_is_written(store, q8):
    spans = [(1, LAYER, 1), (2, LAYER, 1), (3, LAYER // 32, 2), (4, LAYER // 32, 2)] if q8 else \
        [(1, LAYER, 2), (2, LAYER, 2)]
    for i, n, size in spans:
        step = LAYER_AT // (LAYER // n) * size
        for layer in range(LAYERS):
            first = ROOM * i + layer * step
            for spot in (first, first + n * size - 4, first - 4 * N_SEQ + 4, first + n * size // 2):
                store(spot)
