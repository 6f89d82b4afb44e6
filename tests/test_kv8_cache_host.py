"""The arrays of a kv8.Cache (no GPU needed)."""
import pytest
import torch

from pvlc_b200 import kv8


@pytest.mark.parametrize("name", ["codes", "scales", "tails", "table", "tokens", "refs"])
def test_a_cache_keeps_its_tensors(name):
    """The calls go by the addresses that the cache was made with: another tensor in an array's
    place would not be seen, and the first one's memory would be freed under the kernels."""
    c = kv8.Cache.__new__(kv8.Cache)
    t = torch.zeros(4, dtype=torch.int32)
    setattr(c, name, t)
    with pytest.raises(AttributeError, match=name):
        setattr(c, name, t + 1)
    setattr(c, name, getattr(c, name).add_(1))          # as c.tokens += 1 does
    assert getattr(c, name) is t and t.tolist() == [1] * 4
    c.pages = 3
    c.pages = 4
