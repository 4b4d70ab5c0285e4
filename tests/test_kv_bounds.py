"""What the bounds of kv_bounds.py are worth: each is exceeded when one tile of 64 keys, or the sinks, are left out of
the sum (no GPU needed)."""
import pytest
import torch

import kv_bounds as B
from kv_cases import LONG_DECODE, RINGS


def notices(case, hide):
    cache, q, table, L, cu, window, sinks = case
    want, tol = B.attend(cache, q, table, L, cu, window, sinks)
    got, _ = B.attend(cache, q, table, L, cu, window, sinks, hide=hide)
    return bool(((got - want).abs() > tol).any())


@pytest.mark.parametrize("new,lens,H,Hkv,hd,page,window,sinks,dtype,most", LONG_DECODE + RINGS)
def test_a_lost_tile_is_noticed(new, lens, H, Hkv, hd, page, window, sinks, dtype, most):
    cache, q, table, L, cu = B.marked(new[:1], lens[:1], Hkv, Hkv, hd, page, dtype, sinks=sinks)
    one = tuple(x[:, :1].contiguous() for x in cache)  # one head, and the last row of the first sequence
    case = one, q[-1:, :1].contiguous(), table, L, torch.tensor([0, 1], dtype=torch.int32), window, sinks
    low = max(0, lens[0] - window) if window else 0
    tiles = range(low // 64, -(-lens[0] // 64))
    for t in list(tiles)[::max(1, len(tiles) // 40)] + [tiles[0], tiles[-1]]:
        assert notices(case, (64 * t, 64 * t + 64)), t
    if sinks:
        assert notices(case, (0, sinks))
    assert not notices(case, (0, 0))
