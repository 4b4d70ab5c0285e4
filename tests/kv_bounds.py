"""Attention over the paged 8-bit cache from its definition in 64 bits, with a bound that is tight enough to notice a
single lost tile of keys, and inputs whose tiles can be told apart. Test infrastructure, on any device."""
from __future__ import annotations

import math

import torch

import kv_reference as R

F64 = torch.float64
BIAS = 7  # a row's largest weight is 2^BIAS at least when the weights are rounded to fp16
TILE = 64


def attend(cache, q, table, lens, cu, window=0, sinks=0, scale=None, hide=None):
    """(o, bound) in 64 bits; `hide` leaves keys lo .. hi - 1 out. With p the row's softmax, vs the scale and z the bytes
    of a key's values, the weight of a key is w = p vs (up to a factor of the row). The bound counts:
      weights to fp16   2^-11 of each term; of weights below fp16's normals 2^-25 where the row's largest is at least
                        2^BIAS, so 2^-(25 + BIAS) of that one, but no more than the weight itself
      exponents         the score's sum of hd products in fp32, its products and the differences from the maximum
                        (some 16 roundings of numbers of their size), exp2, log2 and 1 / vs: 2^-20 in all; once in the
                        numerator, once in the denominator
      sums              two matrix instructions and two additions per tile of 64 keys, and at most 128 to join parts,
                        each off by 2^-23 of the sum of magnitudes
      the result        half a step of q's type"""
    T, H, hd = q.shape
    k, v, ks, vs = cache
    G, page = H // k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(hd) if scale is None else scale
    o = torch.zeros((T, H, hd), dtype=F64, device=q.device)
    tol = torch.zeros_like(o)
    half = torch.finfo(q.dtype).eps / 2
    least = torch.finfo(q.dtype).smallest_normal * half  # half a step of the subnormals
    for b, n in enumerate((cu[1:] - cu[:-1]).tolist()):
        L, at = int(lens[b]), int(cu[b])
        if n <= 0 or L <= 0:
            continue
        K, V = R.tokens(cache, table[b], L)
        VS = vs[table[b, :-(-L // page)].long()].to(F64).repeat_interleave(page, 0)[:L]  # (L, Hkv)
        pos = torch.arange(L - n, L, device=q.device)[:, None]
        key = torch.arange(L, device=q.device)[None]
        see = key <= pos
        if window:
            see &= (key > pos - window) | (key < sinks)
        if hide:
            see = see & ~((key >= hide[0]) & (key < hide[1]))
        for h in range(H):
            g = h // G
            x, kt = q[at:at + n, h].to(F64), K[:, g].t().contiguous()
            s = torch.matmul(x, kt) * scale
            size = (torch.matmul(x.abs(), kt.abs()) * scale * see).amax(-1, keepdim=True)
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(-1, keepdim=True).clamp(min=-1e300)
            p = torch.exp(s - top)
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            val = V[:, g].contiguous()
            w = p * VS[:, g]
            lost = torch.minimum(w, 2.0 ** -(25 + BIAS) * w.amax(-1, keepdim=True)) * see
            z = val.abs() / VS[:, g, None].clamp(min=1e-300)
            y, spread = torch.matmul(p, val), torch.matmul(p, val.abs())
            logs = VS[:, g].clamp(min=2.0 ** -90).log().abs().max()
            delta = (hd + 8) * 2.0 ** -24 * size + 16 * 2.0 ** -24 * (1 + top.abs() + logs) + 2.0 ** -20
            sums = (4 * (L // TILE + 1) + 128) * 2.0 ** -23
            rel = 2.0 ** -11 + 2 * delta + sums
            o[at:at + n, h] = y
            tol[at:at + n, h] = 1.01 * (half * y.abs() + rel * spread + torch.matmul(lost, z.contiguous())) + least
    return o, tol


def marked(new, lens, H, Hkv, hd, page, dtype, dev="cpu", seed=0, sinks=0):
    """A problem whose weights are of one size (exp of +-0.3 or so) and whose values say where they lie: those of keys
    64 t .. 64 t + 63 are loud in dimension t % hd alone, those of the first `sinks` in the last one."""
    g = torch.Generator().manual_seed(seed)
    table, pages = R.make_table(lens, page, g, "cpu")
    k, v, ks, vs = R.make_cache(pages, Hkv, hd, page, g, "cpu")
    v.zero_()
    for b, L in enumerate(lens):
        for t in range(-(-L // TILE)):
            for at in range(t * TILE, min(L, (t + 1) * TILE)):
                d = hd - 1 if at < sinks else t % hd
                v[table[b, at // page], :, d, at % page] = 100
    q = (0.1 * torch.randn((sum(new), H, hd), generator=g)).to(dtype)
    to = lambda x: x.to(dev)
    return tuple(map(to, (k, v, ks, vs))), to(q), to(table), R.ints(lens, dev), R.cumulative(new, dev)


def sink(new, L, H, Hkv, hd, page, dtype, ahead, loud, dev="cpu", seed=0):
    """One sequence whose first key is `ahead` nats before a flat rest, with values of 0 on a page whose scale is `loud`
    times the others': the output is the rest's, whose weights are small."""
    g = torch.Generator().manual_seed(seed)
    table, pages = R.make_table([L], page, g, "cpu")
    k, v, ks, vs = R.make_cache(pages, Hkv, hd, page, g, "cpu", spread=0.0)
    k.copy_(torch.randint(-2, 3, k.shape, generator=g))
    v.copy_(torch.randint(60, 128, v.shape, generator=g))
    first = table[0, 0]
    k[first, :, 0], v[first, :, :, 0] = 127, 0
    vs[first] *= loud
    x = 1 + 0.1 * torch.randn((new, H, hd), generator=g)
    x = x / x.sum(-1, keepdim=True) * ahead * math.sqrt(hd) / (127 * ks[0, 0])
    to = lambda x: x.to(dev)
    return tuple(map(to, (k, v, ks, vs))), to(x.to(dtype)), to(table), R.ints([L], dev), R.cumulative([new], dev)
