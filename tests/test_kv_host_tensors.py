"""A cache in host memory, with every other argument in order and beside it, is refused before its addresses reach a GPU
(no GPU needed)."""
import pytest
import torch

BF = torch.bfloat16


def test_a_cache_in_host_memory_is_refused():
    from uwc_amd import kv
    cache = kv.new_cache(4, 2, 64, 16, "cpu")
    i = lambda *s: torch.zeros(s, dtype=torch.int32)
    cos = torch.zeros((4, 64))
    with pytest.raises(AssertionError, match="kv.append: the cache must be on a GPU"):
        kv.append(cache, torch.zeros((1, 512), dtype=BF), i(1, 2), i(1), cos, cos)
    with pytest.raises(AssertionError, match="kv.attend: the cache must be on a GPU"):
        kv.attend(cache, torch.zeros((1, 4, 64), dtype=BF), i(1, 2), i(1))
    with pytest.raises(AssertionError, match="kv.read: the cache must be on a GPU"):
        kv.read(cache, i(1, 2), i(1), i(2), 1)
