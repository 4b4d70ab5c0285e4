"""Page table entries below -1, in every form of the attention kernels: a page that is needed and named by no entry of
[0, pages) makes the rows that need it NaN and no others; one that no row needs may be anything."""
import pytest
import torch

import kv_bounds as B

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16

FORMS = [  # new, L, H, Hkv, hd, max_len: 16 rows, 32 rows, four waves, eight waves; in one part, and split
    (1, 500, 4, 2, 64, 1), (1, 3000, 4, 2, 128, 3000), (5, 500, 8, 2, 64, 1 << 22), (80, 500, 4, 2, 64, 1 << 20),
    (80, 2500, 8, 1, 128, 1 << 20), (300, 2000, 4, 1, 128, 20000), (300, 2500, 4, 1, 128, 1 << 20),
]


@pytest.mark.parametrize("new,L,H,Hkv,hd,most", FORMS)
@pytest.mark.parametrize("entry", [-1, -2, -3, -2 ** 31])
def test_attend_needs_a_page_that_no_entry_names(dev, new, L, H, Hkv, hd, most, entry):
    from uwc_amd import kv
    cache, q, table, lens, cu = B.marked([new, new], [L, L - 7], H, Hkv, hd, 16, BF, dev)
    want, tol = B.attend(cache, q, table, lens, cu)
    table[0, (L - new) // 32] = entry  # a page that all of its sequence's rows see
    got = kv.attend(cache, q, table, lens, cu=cu, max_new=new, max_len=most)
    assert torch.isnan(got[:new]).all()
    assert ((got[new:].double() - want[new:]).abs() <= tol[new:]).all()


@pytest.mark.parametrize("new,L,H,Hkv,hd,most", FORMS)
@pytest.mark.parametrize("entry", [-2, -2 ** 31])
def test_attend_does_not_need_a_page_outside_the_window(dev, new, L, H, Hkv, hd, most, entry):
    from uwc_amd import kv
    cache, q, table, lens, cu = B.marked([new], [L], H, Hkv, hd, 16, HF, dev, sinks=5)
    want, tol = B.attend(cache, q, table, lens, cu, 40, 5)
    table[0, 1:(L - new - 40) // 16] = entry
    got = kv.attend(cache, q, table, lens, cu=cu, max_new=new, max_len=most, window=40, sinks=5)
    assert ((got.double() - want).abs() <= tol).all()
