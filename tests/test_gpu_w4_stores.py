"""Linears with 4-bit weights: every form of the kernels with and without a bias, rows of outputs that leave eight, four and one at a
time, and sums of several rounds with a ragged end, against the definition in 64 bits."""
import pytest
import torch

import w4_reference as R
from test_gpu_w4 import rows

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16

# rows, outputs, K of each form for 256 compute units: outputs a multiple of 8, of 4, and neither; where K is long a tile's codes and scales
# are replaced several times, the last time by fewer groups
TILES = [(4096, 4096, 1056), (4001, 4092, 1120), (4000, 4090, 1056),   # 256 x 256
         (2048, 4096, 800), (1030, 4100, 640), (2000, 4090, 1056),     # 128 x 256
         (1024, 4096, 4064), (1000, 4092, 4096), (1000, 4091, 2080),   # 128 x 128
         (512, 4096, 2080), (333, 4092, 2080), (333, 4090, 4128),      # 64 x 128
         (60, 4000, 1056), (60, 3996, 2080), (64, 4003, 1056)]         # 64 x 64
FEW = [(257, 304, 544), (250, 300, 544), (13, 1000, 416), (7, 516, 160), (100, 512, 1024),
       (13, 6200, 160), (3, 6204, 544), (16, 16400, 544), (5, 16388, 96), (2, 16389, 96)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("M,N,K", TILES + FEW)
def test_linear(dev, M, N, K, with_bias, dtype):
    from uwc_amd import w4
    g = torch.Generator().manual_seed(M * 3 + N + K)
    codes, scales = (t.to(dev) for t in R.weight(N, K, g))
    x = rows(M, K, g, dtype, dev)
    bias = (20 * torch.randn(N, generator=g)).to(dtype).to(dev) if with_bias else None
    y = w4.linear(x, codes, scales, bias)
    want, bound = R.linear(x, codes, scales, bias)
    assert ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,F,K", [(4096, 2048, 1056), (4001, 2044, 1120), (4000, 2045, 1056), (700, 4096, 1056), (700, 4092, 1056),
                                   (1024, 2048, 4064), (512, 4092, 2080), (512, 2048, 2080), (333, 2044, 2080), (60, 4000, 1056),
                                   (60, 4004, 2080), (16, 16400, 544), (3, 16388, 544), (40, 304, 9056)])
def test_gated(dev, M, F, K, dtype):
    from uwc_amd import w4
    g = torch.Generator().manual_seed(M * 3 + F + K)
    codes, scales = (t.to(dev) for t in R.weight(2 * F, K, g, 108, 122))
    x = rows(M, K, g, dtype, dev)
    h = w4.gated(x, codes, scales)
    want, bound = R.gated(x, codes, scales)
    assert ((h.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("M,N,K", [(4096, 4096, 160), (2048, 4096, 160), (1024, 4096, 2048), (512, 4096, 1024), (60, 4000, 1056), (257, 304, 544),
                                   (13, 1000, 416)])
def test_outputs_that_begin_at_8_bytes(dev, M, N, K):
    """The C-ABI takes y at any multiple of 8 bytes: the same bits, and nothing beside them."""
    from uwc_amd import _lib, w4
    g = torch.Generator().manual_seed(M + N)
    codes, scales = (t.to(dev) for t in R.weight(N, K, g))
    x, bias = rows(M, K, g, BF, dev), torch.randn(N, generator=g).to(BF).to(dev)
    for b in (bias, None):
        y = torch.full((M * N + 64,), 7.0, dtype=BF, device=dev)
        _lib.call("uwc_w4_linear", x.data_ptr(), K, 0, M, codes.data_ptr(), scales.data_ptr(), N, K, None if b is None else b.data_ptr(),
                  y[36:].data_ptr(), _lib.stream())
        assert (y[:36] == 7).all() and (y[36 + M * N:] == 7).all()
        assert torch.equal(y[36:36 + M * N].view(M, N), w4.linear(x, codes, scales, b))
