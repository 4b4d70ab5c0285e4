"""Linears with 4-bit weights (uwc_amd.w4) on the GPU against the definition in 64 bits."""
import pytest
import torch

import w4_reference as R

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16

# rows: 1, below and past every tile's rows; outputs: below a tile, past one, odd; K: one group, part of a block of 128, more
SHAPES = [(1, 1, 32), (1, 16, 64), (1, 257, 2048), (2, 33, 96), (3, 100, 4096), (7, 515, 160), (16, 64, 256), (17, 48, 1024), (32, 1000, 416),
          (33, 130, 2080), (64, 96, 512), (65, 257, 320), (100, 514, 1024), (128, 256, 2048), (200, 100, 128), (257, 300, 544), (300, 1111, 256),
          (513, 260, 96), (1000, 1030, 1056), (2049, 520, 160), (1030, 4100, 640), (4097, 1026, 384)]
# every form that the rules choose: the tiles of 256 x 256 to 64 x 64 with one, two and four groups of waves, and of few rows
# those for many weights
FORMS = [(4096, 4096, 160), (4001, 4040, 224), (2048, 4096, 160), (2001, 4090, 96), (1024, 4096, 4096), (1000, 4090, 4064), (512, 4096, 2048),
         (333, 4096, 4096), (500, 4001, 2080), (64, 4096, 1024), (60, 4001, 1056), (5, 16400, 96), (3, 6200, 160), (16, 20000, 544), (2, 9300, 288),
         (40, 300, 9056)]


def rows(M, K, g, dtype, dev):
    return (torch.randn((M, K), generator=g) * torch.exp(torch.randn(K, generator=g))).to(dtype).to(dev)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N,K", SHAPES + FORMS)
def test_linear(dev, M, N, K, dtype):
    from uwc_amd import w4
    g = torch.Generator().manual_seed(M * 7 + N + K)
    codes, scales = (t.to(dev) for t in R.weight(N, K, g))
    x = rows(M, K, g, dtype, dev)
    bias = torch.randn(N, generator=g).to(dtype).to(dev) if N % 2 else None
    y = w4.linear(x, codes, scales, bias)
    want, bound = R.linear(x, codes, scales, bias)
    assert y.shape == (M, N) and y.dtype == dtype
    assert ((y.double() - want).abs() <= bound).all()
    assert torch.equal(y, w4.linear(x, codes, scales, bias))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,F,K", [(M, (N + 1) // 2, K) for M, N, K in SHAPES + FORMS])
def test_gated(dev, M, F, K, dtype):
    from uwc_amd import w4
    g = torch.Generator().manual_seed(M * 5 + F + K)
    codes, scales = (t.to(dev) for t in R.weight(2 * F, K, g, 108, 122))
    x = rows(M, K, g, dtype, dev)
    h = w4.gated(x, codes, scales)
    want, bound = R.gated(x, codes, scales)
    assert h.shape == (M, F) and h.dtype == dtype
    assert ((h.double() - want).abs() <= bound).all()
    assert torch.equal(h, w4.gated(x, codes, scales))


@pytest.mark.parametrize("M", [1, 20, 40, 300, 1024])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_every_code_in_every_place(dev, M, dtype):
    """Rows of the identity pick single weights: bit for bit the values, for each place of a block of 128 k."""
    from uwc_amd import w4
    K, N = 320, 272
    n = torch.arange(N)[:, None]
    codes = ((n * 5 + torch.arange(K // 2) * 7) % 256).to(torch.uint8).to(dev)
    scales = (104 + (n * 3 + torch.arange(K // 32)) % 30).to(torch.uint8).to(dev)
    W = R.values(codes, scales)
    for k0 in range(0, K, M):
        x = torch.zeros((M, K), dtype=dtype, device=dev)
        m = min(M, K - k0)
        x[torch.arange(m), k0 + torch.arange(m)] = 1
        y = w4.linear(x, codes, scales)
        assert torch.equal(y[:m].double(), W[:, k0:k0 + m].t()) and not y[m:].any()


def test_extreme_scales(dev):
    """bf16: every scale from 0 to 254 meets its row exactly, as far as fp32 holds the products; 255 is not a number."""
    from uwc_amd import w4
    codes = torch.full((256, 16), 0x21, dtype=torch.uint8, device=dev)  # 0.5, 1
    scales = torch.arange(256, dtype=torch.int32).to(torch.uint8)[:, None].to(dev)
    power = torch.tensor([2.0 ** (i - 127) for i in range(256)], dtype=torch.float64, device=dev)  # pow on a GPU may round
    for M in (1, 300):
        x = torch.zeros((M, 32), dtype=BF, device=dev)
        x[:, 1] = 1
        y = w4.linear(x, codes, scales)[0]
        assert torch.equal(y[1:255].double(), power[1:255]) and torch.isnan(y[255])
        x[:, 1], x[:, 0] = 0, 2.0 ** 100
        y = w4.linear(x, codes, scales)[0]
        assert torch.equal(y[:155].double(), power[:155] * 2.0 ** 99) and torch.isnan(y[255])


@pytest.mark.parametrize("M", [1, 33, 400, 1024])
def test_infinities_and_nan_stay_in_their_rows(dev, M):
    from uwc_amd import w4
    g = torch.Generator().manual_seed(3)
    codes, scales = (t.to(dev) for t in R.weight(300, 256, g))
    scales[7, 3] = 255
    x = rows(M, 256, g, BF, dev)
    clean = w4.linear(x, codes, scales)
    assert torch.isnan(clean[:, 7]).all() and torch.isfinite(clean).sum() == M * 299
    if M > 1:
        x[M // 2, 100] = float("nan")
        y = w4.linear(x, codes, scales)
        keep = torch.arange(M, device=dev) != M // 2
        assert torch.isnan(y[M // 2]).all() and torch.equal(y[keep].nan_to_num(), clean[keep].nan_to_num())
    big = torch.full((M, 256), 3e38, dtype=BF, device=dev)
    six = torch.full((4, 128), 0x77, dtype=torch.uint8, device=dev)
    ones = torch.full((4, 8), 127, dtype=torch.uint8, device=dev)
    assert torch.isinf(w4.linear(big, six, ones)).all()
    assert (w4.gated(-x.abs().nan_to_num() * 100, six, ones) == 0).all()  # silu of far negative numbers


@pytest.mark.parametrize("M", [1, 5, 40, 600])
def test_strides_views_and_shapes(dev, M):
    from uwc_amd import w4
    g = torch.Generator().manual_seed(5)
    codes, scales = (t.to(dev) for t in R.weight(96, 128, g))
    base = rows(M, 400, g, BF, dev)
    dense = base[:, 8:136].contiguous()
    y = w4.linear(dense, codes, scales)
    assert torch.equal(w4.linear(base[:, 8:136], codes, scales), y)  # aligned rows inside wider ones
    odd = torch.empty((M, 400), dtype=BF, device=dev)
    odd[:, 3:131] = dense
    assert torch.equal(w4.linear(odd[:, 3:131], codes, scales), y)  # rows that are not aligned
    assert torch.equal(w4.linear(dense.t().contiguous().t(), codes, scales), y)
    assert torch.equal(w4.linear(dense.view(1, M, 1, 128), codes, scales), y.view(1, M, 1, 96))
    assert torch.equal(w4.linear(dense[0], codes, scales), w4.linear(dense[:1], codes, scales)[0])
    assert torch.equal(w4.linear(dense[:1].expand(M, 128), codes, scales), w4.linear(dense[:1].repeat(M, 1), codes, scales))
    assert torch.equal(w4.linear(dense, codes[16:64], scales[16:64]), y[:, 16:64])  # some rows of a weight
    assert w4.linear(dense[:0], codes, scales).shape == (0, 96) and w4.gated(dense[:0], codes, scales).shape == (0, 48)
    assert w4.linear(dense, codes[:0], scales[:0]).shape == (M, 0)


def test_nothing_outside_the_output_is_written(dev):
    from uwc_amd import _lib, w4
    g = torch.Generator().manual_seed(6)
    for M, N, K in ((1, 17, 64), (5, 33, 96), (40, 70, 160), (300, 259, 256), (1025, 515, 128)):
        codes, scales = (t.to(dev) for t in R.weight(2 * N, K, g))
        x = rows(M, K, g, BF, dev)
        y = torch.full((M * N + 64,), 7.0, dtype=BF, device=dev)
        _lib.call("uwc_w4_linear", x.data_ptr(), K, 0, M, codes.data_ptr(), scales.data_ptr(), N, K, None, y[32:].data_ptr(), _lib.stream())
        assert (y[:32] == 7).all() and (y[32 + M * N:] == 7).all()
        assert torch.equal(y[32:32 + M * N].view(M, N), w4.linear(x, codes[:N], scales[:N]))
        y.fill_(7)
        _lib.call("uwc_w4_gated", x.data_ptr(), K, 0, M, codes.data_ptr(), scales.data_ptr(), N, K, y[32:].data_ptr(), _lib.stream())
        assert (y[:32] == 7).all() and (y[32 + M * N:] == 7).all()
        assert torch.equal(y[32:32 + M * N].view(M, N), w4.gated(x, codes, scales))


@pytest.mark.parametrize("M", [1, 24, 1000])
def test_streams_and_graphs(dev, M):
    """Captured once and replayed on new rows, other eager work between: each replay equals the eager result."""
    from uwc_amd import w4
    g = torch.Generator().manual_seed(8)
    codes, scales = (t.to(dev) for t in R.weight(1024, 512, g))
    x = rows(M, 512, g, BF, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = w4.gated(x, codes, scales), w4.linear(x, codes, scales)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = w4.gated(x, codes, scales), w4.linear(x, codes, scales)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        x.copy_(rows(M, 512, g, BF, dev))
        want = w4.gated(x, codes, scales), w4.linear(x, codes, scales)
