"""uwc_amd.w4 without a GPU: quantization, the values that codes stand for, refusals in Python and at the C-ABI."""
import ctypes
import math

import pytest
import torch

import w4_reference as R

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [torch.float32, BF, HF])
@pytest.mark.parametrize("N,K", [(1, 32), (5, 96), (64, 256)])
def test_quantize_takes_the_nearest_values(dtype, N, K):
    from uwc_amd import w4
    g = torch.Generator().manual_seed(N + K)
    w = (torch.randn((N, K), generator=g) * torch.exp(torch.randn((N, 1), generator=g))).to(dtype)
    w[0, :32] = 0
    codes, scales = w4.quantize(w)
    assert codes.shape == (N, K // 2) and scales.shape == (N, K // 32)
    got = w4.values(codes, scales, torch.float64)
    assert torch.equal(got, R.values(codes, scales))
    for n in range(N):
        for k in range(0, K, 32):
            x = [float(v) for v in w[n, k:k + 32]]
            top = max(map(abs, x))
            e = math.frexp(top)[1] - 3 if top else -127
            assert int(scales[n, k // 32]) == e + 127
            for i, v in enumerate(x):
                best = min(abs(abs(v) - m * 2.0 ** e) for m in R.MAGNITUDES)
                q = float(got[n, k + i])
                assert abs(abs(v) - abs(q)) == best and (q == 0 or (q < 0) == (v < 0))


def test_quantize_ties_and_extremes():
    from uwc_amd import w4
    w = torch.zeros((1, 64))
    w[0, :9] = torch.tensor([7.9, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0])
    w[0, 32:34] = torch.tensor([3.0e38, 1e-45])
    codes, scales = w4.quantize(w)
    v = w4.values(codes, scales, torch.float64)[0]
    assert v[:9].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -4.0] and scales[0, 0] == 127
    assert v[32].item() == 6.0 * 2.0 ** 125 and v[33] == 0
    tiny = torch.full((1, 32), 2.0 ** -130)
    codes, scales = w4.quantize(tiny)
    assert scales[0, 0] == 0 and w4.values(codes, scales).abs().max() == 0  # an eighth of the smallest scale's step
    assert torch.isnan(w4.values(torch.zeros((1, 16), dtype=torch.uint8), torch.full((1, 1), 255, dtype=torch.uint8))).all()


@pytest.mark.parametrize("w", [torch.zeros((2, 33)), torch.zeros(64), torch.zeros((2, 64), dtype=torch.int32), torch.zeros((2, 0)),
                               torch.full((1, 32), float("inf")), torch.full((1, 32), float("nan"))])
def test_quantize_refuses(w):
    from uwc_amd import w4
    with pytest.raises(AssertionError, match="w4.quantize"):
        w4.quantize(w)


U8 = torch.uint8


@pytest.mark.parametrize("change,msg", [
    (dict(x=torch.zeros((2, 64))), "x must be"), (dict(x=torch.zeros((2, 96), dtype=BF)), "x must be"),
    (dict(x=torch.zeros((), dtype=BF)), "x must be"),
    (dict(codes=torch.zeros((4, 32), dtype=torch.int8)), "must be uint8"), (dict(codes=torch.zeros(32, dtype=U8)), "must be uint8"),
    (dict(scales=torch.zeros((4, 2))), "must be uint8"), (dict(scales=torch.zeros((4, 3), dtype=U8)), "positive multiple of 32"),
    (dict(scales=torch.zeros((3, 2), dtype=U8)), "positive multiple of 32"),
    (dict(codes=torch.zeros((4, 24), dtype=U8)), "positive multiple of 32"),
    (dict(codes=torch.zeros((4, 0), dtype=U8), scales=torch.zeros((4, 0), dtype=U8)), "positive multiple of 32"),
    (dict(codes=torch.zeros((32, 4), dtype=U8).t()), "contiguous"),
    (dict(codes=torch.zeros(4 * 32 + 1, dtype=U8)[1:].view(4, 32)), "16-byte aligned"),
    ({}, "on a GPU"),
])
def test_linear_and_gated_refuse(change, msg):
    from uwc_amd import w4
    a = dict(x=torch.zeros((2, 64), dtype=BF), codes=torch.zeros((4, 32), dtype=U8), scales=torch.zeros((4, 2), dtype=U8))
    a.update(change)
    for fn in (w4.linear, w4.gated):
        with pytest.raises(AssertionError, match=msg):
            fn(**a)


FAKE = ctypes.c_void_p(1 << 20)


@pytest.mark.parametrize("change,msg", [
    (dict(dtype=2), b"dtype"), (dict(M=-1), b"bad M"), (dict(N=-1), b"bad M"), (dict(K=0), b"multiple of 32"), (dict(K=48), b"multiple of 32"),
    (dict(K=-32), b"multiple of 32"), (dict(x=None), b"null"), (dict(codes=None), b"null"), (dict(scales=None), b"null"), (dict(y=None), b"null"),
    (dict(stride=68), b"aligned"), (dict(stride=-64), b"aligned"), (dict(x=ctypes.c_void_p((1 << 20) + 8)), b"aligned"),
    (dict(codes=ctypes.c_void_p((1 << 20) + 4)), b"aligned"), (dict(y=ctypes.c_void_p((1 << 20) + 2)), b"aligned"),
    (dict(M=2 ** 31 - 1, N=2 ** 29), b"too many"),
])
def test_the_library_refuses(change, msg):
    from uwc_amd import _lib
    L = _lib.lib()
    a = dict(x=FAKE, stride=64, dtype=0, M=1, codes=FAKE, scales=FAKE, N=16, K=64, bias=None, y=FAKE)
    a.update(change)
    assert L.uwc_w4_linear(*a.values(), None) == -1 and msg in L.uwc_last_error()
    del a["bias"]
    assert L.uwc_w4_gated(*a.values(), None) == -1 and msg in L.uwc_last_error()


def test_nothing_to_do_is_no_error():
    from uwc_amd import _lib
    L = _lib.lib()
    for M, N in ((0, 16), (4, 0)):
        assert L.uwc_w4_linear(None, 64, 0, M, None, None, N, 64, None, None, None) == 0
        assert L.uwc_w4_gated(None, 64, 0, M, None, None, N, 64, None, None) == 0
