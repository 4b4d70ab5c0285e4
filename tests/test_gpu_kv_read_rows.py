"""Reading the paged 8-bit cache back writes every row of its outputs: rows of no sequence are zeros, those of a sequence that
starts before its first token NaN, whatever the outputs held."""
import math

import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def read(cache, table, start, cu, rows, dtype):
    """uwc_kv_read into buffers that hold sevens, with a guard row behind."""
    from uwc_amd import _lib
    k, v, ks, vs = cache
    pages, Hkv, page, hd = k.shape
    out = [torch.full((rows + 1, Hkv, hd), 7, dtype=dtype, device=k.device) for _ in range(2)]
    _lib.call("uwc_kv_read", k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, page, Hkv, hd, table.data_ptr(),
              table.stride(0), table.shape[1], start.data_ptr(), cu.data_ptr(), len(start), rows, 0 if dtype == BF else 1,
              out[0].data_ptr(), out[1].data_ptr(), _lib.stream())
    for x in out:
        assert (x[rows] == 7).all()
    return [x[:rows] for x in out]


def expect(cache, table, start, cu, rows, dtype):
    k, v, ks, vs = cache
    out = [torch.zeros((rows, k.shape[1], k.shape[3]), dtype=dtype, device=k.device) for _ in range(2)]
    for b in range(len(start)):
        lo, hi, s = int(cu[b]), int(cu[b + 1]), int(start[b])
        if s < 0:
            for x in out:
                x[lo:hi] = math.nan
            continue
        pos = torch.arange(s, s + hi - lo, device=k.device)
        pg, slot = table[b, pos // k.shape[2]].long(), pos % k.shape[2]
        out[0][lo:hi] = (k[pg, :, slot].float() * ks[pg][..., None]).to(dtype)
        out[1][lo:hi] = (v[pg, :, :, slot].float() * vs[pg][..., None]).to(dtype)
    return out


# the third: a sequence of 2 tokens in two pages of 16 and a rest of less than a page
@pytest.mark.parametrize("n,start,page", [([1, 0, 65, 200], [129, 3, 0, 17], 64), ([5], [0], 128), ([2], [15], 16), ([33, 2, 18], [30, 31, 15], 32),
                                          ([0, 0], [4, 0], 16)])
@pytest.mark.parametrize("pad", [0, 1, 13, 64, 1001])
@pytest.mark.parametrize("Hkv,hd,dtype", [(2, 64, BF), (3, 128, HF), (1, 32, BF)])
def test_rows_of_no_sequence_are_zeros(dev, n, start, page, pad, Hkv, hd, dtype):
    g = torch.Generator().manual_seed(len(n) + pad)
    table, pages = R.make_table([a + b for a, b in zip(n, start)], page, g, dev)
    cache = R.make_cache(pages, Hkv, hd, page, g, dev)
    args = cache, table, R.ints(start, dev), R.cumulative(n, dev), sum(n) + pad, dtype
    for got, want in zip(read(*args), expect(*args)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("start", [-1, -5, -64, -2 ** 31])
@pytest.mark.parametrize("page", [16, 64])
def test_a_negative_start_is_not_a_number(dev, start, page):
    g = torch.Generator().manual_seed(1)
    n = [9, 130, 0, 40]
    table, pages = R.make_table([a + 20 for a in n], page, g, dev)
    cache = R.make_cache(pages, 2, 64, page, g, dev)
    args = cache, table, R.ints([3, start, start, 17], dev), R.cumulative(n, dev), sum(n) + 50, HF
    for got, want in zip(read(*args), expect(*args)):
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_no_sequence_at_all(dev):
    from uwc_amd import kv
    cache = kv.new_cache(2, 2, 64, 16, dev)
    table = torch.zeros((0, 3), dtype=torch.int32, device=dev)
    for x in read(cache, table, R.ints([], dev), R.ints([0], dev), 70, BF):
        assert not x.any()
    for x in kv.read(cache, table, R.ints([], dev), R.ints([0], dev), 70):
        assert x.shape == (70, 2, 64) and not x.any()
