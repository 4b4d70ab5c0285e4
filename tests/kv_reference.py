"""The paged 8-bit key/value cache's operators from their definitions, in 64 bits, with the bounds that the
kernels' roundings allow. Test infrastructure: one sequence and one head at a time, on any device."""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def cumulative(n, dev):
    t = torch.zeros(len(n) + 1, dtype=torch.int32)
    t[1:] = torch.tensor(n, dtype=torch.int64).cumsum(0)
    return t.to(dev)


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def make_table(lens, page, g, dev, spare=3, width=None):
    """Shuffled pages for sequences of these lengths: (table with -1 past a sequence's pages, pages in all)."""
    held = [-(-n // page) for n in lens]
    width = max(held + [1]) if width is None else width
    order = torch.randperm(sum(held) + spare, generator=g).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(dev), sum(held) + spare


def make_cache(pages, Hkv, hd, page, g, dev, spread=0.4):
    q = lambda *s: torch.clamp(torch.round(30 * torch.randn(s, generator=g)), -127, 127).to(torch.int8).to(dev)
    s = lambda: (torch.exp(spread * torch.randn((pages, Hkv), generator=g)) / 30).to(dev)
    return q(pages, Hkv, page, hd), q(pages, Hkv, hd, page), s(), s()


def tokens(cache, row, n):
    """Keys and values of a sequence's first n tokens, (n, Hkv, hd) in 64 bits."""
    k, v, ks, vs = cache
    page = k.shape[2]
    ids = row[:-(-n // page)].long()
    K = (k[ids].to(F64) * ks[ids].to(F64)[..., None, None]).transpose(1, 2)
    V = (v[ids].to(F64) * vs[ids].to(F64)[..., None, None]).permute(0, 3, 1, 2)
    return K.reshape(-1, *K.shape[2:])[:n], V.reshape(-1, *V.shape[2:])[:n]


def attend(cache, q, table, lens, cu, window=0, sinks=0, scale=None):
    """(o, bound) in 64 bits. The bound counts the kernels' roundings: probabilities to fp16 (2^-11 of each
    term, 2^-25 below fp16's normals, of weights at most the row's largest), scores summed in fp32 (hd + 8
    roundings of 2^-24 of the sum of magnitudes, in the exponent), exponentials and sums in fp32, and the
    result to q's type."""
    T, H, hd = q.shape
    G = H // cache[0].shape[1]
    scale = 1 / math.sqrt(hd) if scale is None else scale
    o = torch.zeros((T, H, hd), dtype=F64, device=q.device)
    tol = torch.zeros_like(o)
    half = torch.finfo(q.dtype).eps / 2
    for b, n in enumerate((cu[1:] - cu[:-1]).tolist()):
        L, at = int(lens[b]), int(cu[b])
        if n <= 0 or L <= 0:
            continue
        K, V = tokens(cache, table[b], L)
        pos = torch.arange(L - n, L, device=q.device)[:, None]
        key = torch.arange(L, device=q.device)[None]
        see = key <= pos
        if window:
            see &= (key > pos - window) | (key < sinks)
        for h in range(H):
            x = q[at:at + n, h].to(F64)
            kt = K[:, h // G].t().contiguous()
            s = torch.matmul(x, kt) * scale
            mag = torch.matmul(x.abs(), kt.abs()) * scale  # sums of magnitudes
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(-1, keepdim=True).clamp(min=-1e300)
            p = torch.exp(s - top)
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            v = V[:, h // G].contiguous()
            o[at:at + n, h] = torch.matmul(p, v)
            spread = torch.matmul(p, v.abs())
            size = (mag * see).amax(-1, keepdim=True)
            delta = (hd + 8) * 2.0 ** -24 * size + 16 * 2.0 ** -24 * (1 + top.abs().clamp(max=1e30)) + 2.0 ** -20
            tol[at:at + n, h] = (half * o[at:at + n, h].abs() + (2.0 ** -11 + 2 * delta + L * 2.0 ** -24) * spread * 1.01
                                 + L * 2.0 ** -25 * v.abs().max() + 2.0 ** -25)
    return o, tol


def norm_turn(x, w, cos, sin, eps):
    """(value, magnitude) of heads x (n, heads, hd) normed and rotated, in 64 bits."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.to(F64)
    lo, hi = x.chunk(2, -1)
    turned = torch.cat([-hi, lo], -1)
    c, s = cos.to(F64)[:, None], sin.to(F64)[:, None]
    return x * c + turned * s, (x * c).abs() + (turned * s).abs()
