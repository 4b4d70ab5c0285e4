"""Without _kv.so, or with one that does not fit this torch, uwc_amd.kv warns once and calls the library through ctypes (no
GPU needed: each call ends at the check that follows all others)."""
import sys
import warnings

import pytest
import torch

BF = torch.bfloat16


def test_calls_go_through_ctypes(monkeypatch):
    import uwc_amd
    from uwc_amd import _lib, kv
    monkeypatch.setattr(_lib, "_KV", None)
    monkeypatch.setitem(sys.modules, "uwc_amd._kv", None)  # the import fails
    monkeypatch.delattr(uwc_amd, "_kv", raising=False)
    cache = kv.new_cache(4, 2, 64, 16, "cpu")
    i = lambda *s: torch.zeros(s, dtype=torch.int32)
    cos = torch.zeros((4, 64))
    with pytest.warns(RuntimeWarning, match="_kv.so is not built or does not fit"):
        with pytest.raises(AssertionError, match="kv.attend: the cache must be on a GPU"):
            kv.attend(cache, torch.zeros((1, 4, 64), dtype=BF), i(1, 2), i(1))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(AssertionError, match="kv.append: the cache must be on a GPU"):
            kv.append(cache, torch.zeros((1, 512), dtype=BF), i(1, 2), i(1), cos, cos)
        with pytest.raises(AssertionError, match="kv.read: the cache must be on a GPU"):
            kv.read(cache, i(1, 2), i(1), i(2), 1)


@pytest.mark.gpu
def test_the_same_bits(dev, monkeypatch):
    import uwc_amd
    from uwc_amd import _lib, kv
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn((3, 8 * 64), generator=g).to(BF).to(dev)
    cos = torch.rand((40, 64), generator=g).to(dev)
    table = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32, device=dev)
    ctx = torch.tensor([0, 15, 20], dtype=torch.int32, device=dev)
    cu = torch.arange(4, dtype=torch.int32, device=dev)

    def step():
        cache = kv.new_cache(6, 2, 64, 16, dev)
        q = kv.append(cache, qkv, table, ctx, cos, cos)
        return (q, kv.attend(cache, q, table, ctx + 1, max_len=21), *kv.read(cache, table, ctx, cu, 3), *cache)

    want = step()
    monkeypatch.setattr(_lib, "_KV", None)
    monkeypatch.setitem(sys.modules, "uwc_amd._kv", None)
    monkeypatch.delattr(uwc_amd, "_kv", raising=False)
    with pytest.warns(RuntimeWarning):
        got = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
