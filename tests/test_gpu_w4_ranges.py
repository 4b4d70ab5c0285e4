"""The range of 4-bit weights: which scales meet rows of either type exactly, what is rounded, what is infinite."""
import pytest
import torch

import w4_reference as R

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def one_weight_a_row(dev, K=32):
    """A weight of 16 x 256 rows: code c at scale s in column 1, zeros beside it; and its values, in 64 bits."""
    c, s = torch.meshgrid(torch.arange(16), torch.arange(256), indexing="ij")
    codes = torch.zeros((4096, K // 2), dtype=torch.uint8)
    codes[:, 0] = (16 * c.flatten()).to(torch.uint8)
    scales = s.flatten()[:, None].repeat(1, K // 32).to(torch.uint8)
    return codes.to(dev), scales.to(dev), R.values(codes[:, :16], scales[:, :1])[:, 1].to(dev), s.flatten().to(dev)


@pytest.mark.parametrize("M", [1, 300])
@pytest.mark.parametrize("K", [32, 256])
@pytest.mark.parametrize("power", [-100, 0, 100])
def test_bfloat16(dev, M, K, power):
    """Exact for scales up to 252, and above for every value below 2^128; others are infinite, and their outputs no numbers. Rows of
    2^power bring outputs into fp32's normal range."""
    from uwc_amd import w4
    codes, scales, w, s = one_weight_a_row(dev, K)
    x = torch.zeros((M, K), dtype=BF, device=dev)
    x[:, 1] = 2.0 ** power
    y = w4.linear(x, codes, scales)
    want = w * 2.0 ** power
    held = (w.abs() < 2.0 ** 128) & (s < 255)
    assert held[s <= 252].all()
    at = held & (want.abs() < 2.0 ** 128) & ((want.abs() >= 2.0 ** -126) | (w == 0))
    assert at.sum() > 2000 and torch.equal(y[:, at].double(), want[at].expand(M, -1))
    assert not torch.isfinite(y[:, (s < 255) & ~held]).any()
    assert torch.isnan(y[:, s == 255]).all()


@pytest.mark.parametrize("M", [1, 300])
@pytest.mark.parametrize("K", [32, 256])
def test_float16(dev, M, K):
    """Exact for scales from 104 to 140; smaller ones are rounded to fp16's smallest step, 2^-24; what is 65520 and more is infinite."""
    from uwc_amd import w4
    codes, scales, w, s = one_weight_a_row(dev, K)
    x = torch.zeros((M, K), dtype=HF, device=dev)
    x[:, 1] = 1
    y = w4.linear(x, codes, scales).double()
    exact = (s >= 104) & (s <= 140)
    assert torch.equal(y[:, exact], w[exact].expand(M, -1))
    assert ((y - w).abs()[:, s < 104] <= 2.0 ** -25).all()
    held = (s > 140) & (s < 255) & (w.abs() < 65520)
    assert torch.equal(y[:, held], w[held].expand(M, -1))
    assert not torch.isfinite(y[:, (s > 140) & (s < 255) & ~held]).any()
    assert torch.isnan(y[:, s == 255]).all()
    assert not torch.equal(y[0, s == 103], w[s == 103])  # 0.5 and 1.5 have no such step
