"""GPU parity of attention over the paged 8-bit cache where a lost or doubled tile of keys would show: values that mark
their tiles, with the bounds of kv_bounds.py."""
import pytest
import torch

import kv_bounds as B
from kv_cases import LONG_DECODE, RINGS

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def check(got, want, tol, what=""):
    err = (got.double() - want).abs()
    worst = (err - tol).max().item()
    assert not torch.isnan(err).any() and worst <= 0, f"{what}: off by {worst:.3g} more than its bound, {(err / tol).max().item():.3g} of it"


@pytest.mark.parametrize("new,lens,H,Hkv,hd,page,window,sinks,dtype,most", LONG_DECODE + RINGS)
def test_attend_counts_every_tile_once(dev, new, lens, H, Hkv, hd, page, window, sinks, dtype, most):
    from uwc_amd import kv
    cache, q, table, L, cu = B.marked(new, lens, H, Hkv, hd, page, dtype, dev, sinks=sinks)
    want, tol = B.attend(cache, q, table, L, cu, window, sinks)
    args = dict(cu=None if max(new) == 1 else cu, max_new=max(new), max_len=most, window=window, sinks=sinks)
    got = kv.attend(cache, q, table, L, **args)
    check(got, want, tol)
    assert torch.equal(got, kv.attend(cache, q, table, L, **args))
