"""What a paged cache is, apart from its kernels (no GPU)."""
import pytest

from gpt_neox_amd.paged_cache import PagedKVCache


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale", "pages", "page_size", "heads", "dim", "dtype", "device", "quantised"])
def test_what_was_checked_cannot_be_replaced(name):
    # the calls go by the sizes and strides that the constructor has looked at
    cache = object.__new__(PagedKVCache)
    setattr(cache, name, 1)
    with pytest.raises(AttributeError, match="cannot be replaced"):
        setattr(cache, name, 2)
    assert getattr(cache, name) == 1
    cache.label = "layer 3"  # a name of the caller's own
    cache.label = "layer 4"
