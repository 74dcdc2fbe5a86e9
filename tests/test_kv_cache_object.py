"""ops.KvCache keeps the tensors whose addresses it gave to the library (no GPU)."""
import pytest

from sager_amd import ops


@pytest.mark.parametrize("name", ["k", "v", "pages", "length"])
def test_its_tensors_cannot_be_replaced(name):
    """cache.length = cache.commit(...) would leave the kernels with the old lengths' address, and
    their memory to be used for something else: it raises."""
    cache = object.__new__(ops.KvCache)
    kept = object()
    cache._tensors = dict.fromkeys(("k", "v", "pages", "length"), kept)
    assert getattr(cache, name) is kept
    with pytest.raises(AttributeError):
        setattr(cache, name, object())
    assert getattr(cache, name) is kept
