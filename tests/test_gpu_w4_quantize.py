"""w4.quantize on a GPU gives the codes and scales that it gives on the host, numbers below fp32's normal range among them."""
import pytest
import torch

import w4_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16])
def test_the_same_as_on_the_host(dev, dtype):
    from uwc_amd import w4
    g = torch.Generator().manual_seed(5)
    w = torch.randn((300, 96), generator=g, dtype=torch.float64)
    w = w * 2.0 ** (torch.arange(300) - 160)[:, None].clamp(max=100).double()  # from below the smallest scale up
    w = w.to(dtype)
    w = torch.where(torch.isfinite(w), w, torch.zeros_like(w))
    w[0, :32], w[1, 0] = 0, -w[1, 0]
    codes, scales = w4.quantize(w)
    for a, b in zip(w4.quantize(w.to(dev)), (codes, scales)):
        assert torch.equal(a.cpu(), b)
    want = R.values(codes, scales)
    assert torch.equal(w4.values(codes.to(dev), scales.to(dev), torch.float64).cpu(), want)
    assert len(scales.unique()) > 10 and want.abs().max() > 0
