"""A cache without pages, kv heads, tokens or dimensions is refused by every entry of uwc_amd.kv before a size of it divides
anything, on the CPU and, where the native way takes the call first, on a GPU."""
import pytest
import torch

BF = torch.bfloat16


def empty(dim, dev):
    n = [4, 2, 16, 64]
    n[dim] = 0
    z = lambda *s: torch.zeros(s, dtype=torch.int8, device=dev)
    f = lambda: torch.zeros((n[0], n[1]), device=dev)
    return z(*n), z(n[0], n[1], n[3], n[2]), f(), f()


def refuses(dev, dim):
    from uwc_amd import kv
    cache = empty(dim, dev)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)
    q, cos = torch.zeros((1, 4, cache[0].shape[3]), dtype=BF, device=dev), torch.zeros((4, cache[0].shape[3]), device=dev)
    with pytest.raises(AssertionError, match="kv.attend: the cache is empty"):
        kv.attend(cache, q, i(1, 2), i(1))
    with pytest.raises(AssertionError, match="kv.append: the cache is empty"):
        kv.append(cache, torch.zeros((1, 512), dtype=BF, device=dev), i(1, 2), i(1), cos, cos)
    with pytest.raises(AssertionError, match="kv.read: the cache is empty"):
        kv.read(cache, i(1, 2), i(1), i(2), 1)


@pytest.mark.parametrize("dim", range(4))
def test_empty_caches_are_refused(dim):
    refuses("cpu", dim)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", range(4))
def test_empty_caches_are_refused_on_a_gpu(dev, dim):
    refuses(dev, dim)
