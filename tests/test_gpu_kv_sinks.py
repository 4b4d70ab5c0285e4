"""GPU parity of attention over the paged 8-bit cache where one key is far ahead of a long flat rest and has values of
zero: the output is that of small weights. Bounds of kv_bounds.py, derived from the roundings."""
import pytest
import torch

import kv_bounds as B

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16

FORMS = [  # new, L, H, Hkv, hd, max_len: 16 rows in one part and in many, 32 rows, four waves, eight waves, both split
    (1, 4000, 4, 2, 128, 1), (1, 20000, 4, 1, 128, 20000), (5, 9000, 8, 2, 64, 1 << 22), (100, 9000, 4, 1, 64, 1 << 20),
    (100, 9000, 4, 1, 32, 9000 * 16), (300, 9000, 4, 1, 128, 9000), (300, 9000, 4, 1, 128, 1 << 20),
]


@pytest.mark.parametrize("new,L,H,Hkv,hd,most", FORMS)
@pytest.mark.parametrize("ahead,loud,dtype", [(14, 1, HF), (16, 1, BF), (17, 1, HF), (18, 1, BF), (14, 8, BF), (16, 8, HF)])
def test_attend_tail_behind_a_sink(dev, new, L, H, Hkv, hd, most, ahead, loud, dtype):
    from uwc_amd import kv
    cache, q, table, lens, cu = B.sink(new, L, H, Hkv, hd, 16, dtype, ahead, loud, dev)
    want, tol = B.attend(cache, q, table, lens, cu)
    got = kv.attend(cache, q, table, lens, cu=None if new == 1 else cu, max_len=most)
    err = (got.double() - want).abs()
    assert not torch.isnan(err).any() and (err <= tol).all(), f"{(err / tol).max().item():.3g} of the bound, " \
        f"{(err.norm() / want.norm()).item():.3g} of the norm"
