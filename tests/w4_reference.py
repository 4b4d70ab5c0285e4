"""Linears with 4-bit weights from their definition, in 64 bits, with the bounds that the kernels' roundings allow. Test
infrastructure."""
from __future__ import annotations

import torch

F64 = torch.float64
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def weight(N, K, g, low=110, high=124):
    """Random codes and scales on the host."""
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.int32).to(torch.uint8)
    scales = torch.randint(low, high + 1, (N, K // 32), generator=g, dtype=torch.int32).to(torch.uint8)
    return codes, scales


def values(codes, scales):
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), dtype=F64, device=codes.device)
    w = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=F64, device=codes.device)
    w[:, 0::2] = table[(codes % 16).long()]
    w[:, 1::2] = table[(codes // 16).long()]
    powers = torch.tensor([2.0 ** (i - 127) for i in range(256)], dtype=F64, device=codes.device)  # pow on a GPU may round
    return w * powers[scales.long()].repeat_interleave(32, 1)


def linear(x, codes, scales, bias=None):
    """(y, bound): products are exact in fp32. A sum is a chain of K / 32 additions, each of 32 products, and the join
    of at most 16 parts: no more than K / 32 + 32 + 16 roundings of at most 2^-23 of the sum of magnitudes; the
    bias is one more, then half a step of the output's type."""
    X, W = x.reshape(-1, x.shape[-1]).to(F64), values(codes, scales).t().contiguous()
    y, size = torch.matmul(X, W), torch.matmul(X.abs(), W.abs())
    if bias is not None:
        y, size = y + bias.to(F64), size + bias.to(F64).abs()
    acc = (x.shape[-1] / 32 + 50) * 2.0 ** -23 * size
    half = torch.finfo(x.dtype).eps / 2
    bound = acc + half * (y.abs() + acc) + torch.finfo(x.dtype).smallest_normal
    return y.view(*x.shape[:-1], -1), bound.view(*x.shape[:-1], -1)


def gated(x, codes, scales):
    """(h, bound): the projections' errors go through silu (its slope is at most 1.1) and the product; silu itself is off by
    (|g| + 8) 2^-22 of itself (the exponential's argument is rounded once, then three operations)."""
    F = codes.shape[0] // 2
    X, W = x.reshape(-1, x.shape[-1]).to(F64), values(codes, scales).t().contiguous()
    y, size = torch.matmul(X, W), torch.matmul(X.abs(), W.abs())
    d = (x.shape[-1] / 32 + 50) * 2.0 ** -23 * size
    g, u, dg, du = y[:, :F], y[:, F:], d[:, :F], d[:, F:]
    s = g * torch.sigmoid(g)
    ds = 1.1 * dg + s.abs() * (g.abs() + 8) * 2.0 ** -22
    h = s * u
    dh = ds * u.abs() + s.abs() * du + ds * du
    half = torch.finfo(x.dtype).eps / 2
    bound = dh + (half + 2.0 ** -23) * (h.abs() + dh) + torch.finfo(x.dtype).smallest_normal
    return h.view(*x.shape[:-1], F), bound.view(*x.shape[:-1], F)
