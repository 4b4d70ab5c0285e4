"""Linears with 4-bit weights on MI355X, for serving models whose weights' bytes bound every token: the OCP
microscaling format of fp4 elements (the reference's linears are 8-bit, runtime/detrt/qwen3.py:71-126; here
uwc_amd.detrt and uwc_amd.model).

A weight is (codes, scales): codes uint8 (N, K / 2), the weight of column 2 i in the low half of byte i and that of
column 2 i + 1 in the high half, scales uint8 (N, K / 32), one for each group of 32 columns of a row:

    w[n, k] = value(code) 2^(scale - 127)     value = 0, 0.5, 1, 1.5, 2, 3, 4, 6; negated where the code has bit 3

  quantize  the nearest codes and scales of a matrix (once, when a model is loaded)
  values    the matrix that they stand for
  linear    x W^T (+ bias)
  gated     silu(x G^T) * (x U^T): both projections, the activation and the product of a feed-forward block in one kernel

Rows x are bfloat16 or float16, sums fp32, rounded once to x's type. bfloat16 rows meet weights below 2^128 exactly, which all of
scales up to 252 are; for float16 rows the weights are rounded to float16 (exact for scales from 104 to 140). Weights past
those ranges (2^128, and for float16 65520) are infinite, and the outputs that they meet infinite or not a number.
A scale of 255 is not a number: its row's outputs are NaN. Nothing is recorded for autograd.

The same call gives the same bits every time. Which kernel runs, and in how many parts it sums, goes by the number of rows (and N and
K): the same row among others may differ in the last bits, unlike in the framework's integer linears.

Everything runs on torch's current HIP stream; buffers are torch tensors on the caller's GPU. Arguments of the usual form
take the short way of uwc_amd.kv.
"""
from __future__ import annotations

import torch

from . import _lib, kv

_TYPES = {torch.bfloat16: 0, torch.float16: 1}
GROUP = 32
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _powers(device) -> torch.Tensor:
    """2^(i - 127) at i, in 64 bits: exact, which pow on a GPU need not be; not a number at 255."""
    return torch.tensor([2.0 ** (i - 127) for i in range(255)] + [float("nan")], dtype=torch.float64, device=device)


def _require(ok, msg):
    if not ok:
        raise AssertionError(msg)


def quantize(w: torch.Tensor):
    """(codes, scales) of a matrix w (N, K), K a multiple of 32, of finite numbers within float32: a group's scale is the power of
    two, at least 2^-127, that brings its largest magnitude into [4, 8) (an all-zero group's is 2^-127), each weight the nearest
    value, ties to the code with a zero low bit, 6 where it is larger."""
    _require(w.dim() == 2 and w.is_floating_point() and w.shape[1] % GROUP == 0 and w.shape[1] > 0,
             f"w4.quantize: w must be a floating-point (N, K) with K a positive multiple of {GROUP}, got {w.dtype} {tuple(w.shape)}")
    N, K = w.shape
    codes = torch.empty((N, K // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((N, K // GROUP), dtype=torch.uint8, device=w.device)
    powers = _powers(w.device)
    step = max(1, (1 << 25) // K)  # rows at a time: an lm_head never needs a whole fp32 copy
    for n in range(0, N, step):
        x = w[n:n + step].detach()
        x = (x if x.dtype == torch.float64 else x.float()).unflatten(1, (-1, GROUP))
        top = x.abs().amax(-1, keepdim=True)
        _require(bool(torch.isfinite(top.float()).all()), "w4.quantize: w has infinities or NaN")
        e = (torch.frexp(top).exponent - 3).clamp(min=-127)  # top = m 2^(e + 3), m in [0.5, 1)
        e = torch.where(top > 0, e, -127)
        y = x.double().abs() / powers[(e + 127).long()]  # below 8
        # halfway points between neighbours; a tie goes to the even code: up at 0.75, 1.75, 3.5, down at 0.25, 1.25, 2.5, 5
        c = torch.zeros_like(x, dtype=torch.uint8)
        for point, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
            c += (y >= point) if up else (y > point)
        c = (c | ((x < 0).to(torch.uint8) << 3)).view(-1, K // 2, 2)
        codes[n:n + step] = c[..., 0] | (c[..., 1] << 4)
        scales[n:n + step] = (e.squeeze(-1) + 127).to(torch.uint8)
    return codes, scales


def values(codes: torch.Tensor, scales: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """The weights (N, K) that codes and scales stand for."""
    N, K = _weight("w4.values", codes, scales)
    c = torch.stack([codes & 15, codes >> 4], -1).view(N, -1, GROUP)
    v = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64, device=codes.device)[c.long()]
    return (v * _powers(codes.device)[scales.long()].unsqueeze(-1)).view(N, K).to(dtype)


def _weight(fn, codes, scales):
    """(N, K) of a checked weight."""
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2 or scales.dim() != 2:
        raise AssertionError(f"{fn}: codes and scales must be uint8 (N, K / 2) and (N, K / {GROUP}), got {codes.dtype} "
                             f"{tuple(codes.shape)} and {scales.dtype} {tuple(scales.shape)}")
    N, K = codes.shape[0], codes.shape[1] * 2
    if K == 0 or K % GROUP or scales.shape != (N, K // GROUP) or scales.device != codes.device:
        raise AssertionError(f"{fn}: codes (N, K / 2) and scales (N, K / {GROUP}) of one device, K a positive multiple of {GROUP}; "
                             f"got {tuple(codes.shape)} on {codes.device} and {tuple(scales.shape)} on {scales.device}")
    return N, K


def _call(fn, x, codes, scales):
    """(x as rows, N, K) of checked arguments: rows that are not dense and aligned are copied, weights are not."""
    N, K = _weight(fn, codes, scales)
    if x.dtype not in _TYPES or x.device != codes.device or x.dim() < 1 or x.shape[-1] != K:
        raise AssertionError(f"{fn}: x must be bfloat16 or float16 (..., {K}) on the weight's device, got {x.dtype} "
                             f"{tuple(x.shape)} on {x.device}")
    if max(N, K, x.numel() // K) > kv._I32MAX:
        raise AssertionError(f"{fn}: rows, outputs and K must be below 2^31, got {x.numel() // K}, {N} and {K}")
    if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 16:
        raise AssertionError(f"{fn}: codes and scales must be contiguous, codes 16-byte aligned")
    if x.device.type != "cuda":
        raise AssertionError(f"{fn}: the weight must be on a GPU, got {x.device}")
    rows = x.reshape(-1, K)
    if not (rows.stride(1) == 1 and rows.stride(0) % 8 == 0 and 0 <= rows.stride(0) <= 1 << 22 and rows.data_ptr() % 16 == 0):
        rows = rows.clone(memory_format=torch.contiguous_format)
    return rows, N, K


def linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, bias=None) -> torch.Tensor:
    """x W^T (+ bias): (..., N) in x's type, for x (..., K); bias (N,) in x's type."""
    r = _lib.kv().linear(x, codes, scales, bias, kv._stream())
    if r is not None:
        return r if type(r) is not int else _lib.fail("uwc_w4_linear", r)
    fn = "w4.linear"
    rows, N, K = _call(fn, x, codes, scales)
    if bias is not None:
        if bias.dtype != x.dtype or tuple(bias.shape) != (N,) or bias.device != x.device:
            raise AssertionError(f"{fn}: bias must be {x.dtype} ({N},) on x's device, got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
        bias = bias.contiguous()
    with torch.cuda.device(x.device):
        y = torch.empty((rows.shape[0], N), dtype=x.dtype, device=x.device)
        _lib.call("uwc_w4_linear", rows.data_ptr(), rows.stride(0), _TYPES[x.dtype], rows.shape[0], codes.data_ptr(), scales.data_ptr(),
                  N, K, None if bias is None else bias.data_ptr(), y.data_ptr(), _lib.stream())
    return y.view(*x.shape[:-1], N)


def gated(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """silu(x G^T) * (x U^T): (..., F) in x's type; the weight's first F rows are G, the other F are U."""
    r = _lib.kv().gated(x, codes, scales, kv._stream())
    if r is not None:
        return r if type(r) is not int else _lib.fail("uwc_w4_gated", r)
    fn = "w4.gated"
    rows, N, K = _call(fn, x, codes, scales)
    _require(N % 2 == 0, f"{fn}: the weight's rows are a gate's and as many of the other projection, got {N}")
    with torch.cuda.device(x.device):
        y = torch.empty((rows.shape[0], N // 2), dtype=x.dtype, device=x.device)
        _lib.call("uwc_w4_gated", rows.data_ptr(), rows.stride(0), _TYPES[x.dtype], rows.shape[0], codes.data_ptr(), scales.data_ptr(),
                  N // 2, K, y.data_ptr(), _lib.stream())
    return y.view(*x.shape[:-1], N // 2)
