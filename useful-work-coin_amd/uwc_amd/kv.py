"""A paged key/value cache held in 8 bits, and the causal attention that reads it, on MI355X: what a
model of these integer linears needs to generate token by token and to serve several sequences of
different lengths (the reference's generate_greedy keeps whole fp32 rows of one sequence,
runtime/detrt/qwen3.py:296-334).

The cache of one layer is (k, v, ks, vs):
  k   int8 (pages, kv heads, page, head_dim)
  v   int8 (pages, kv heads, head_dim, page), tokens innermost
  ks  fp32 (pages, kv heads): a page's keys of one head are k * ks
  vs  fp32 (pages, kv heads): its values v * vs
page is 16, 32, 64 or 128 tokens, head_dim 32, 64 or 128. Token p of sequence b lies in slot p % page
of page table[b, p // page]; which pages a sequence gets is the caller's to say.

  new_cache   an empty cache
  append      new tokens' heads: norm, rotation, q out, keys and values quantized into their pages
  attend      attention of new queries over the cache, grouped heads, window and sinks
  read        a range of cached tokens as values

The new tokens of several sequences are packed along the first axis: sequence b's are rows
cu[b] .. cu[b + 1] - 1 (int32, cu[0] = 0); without cu every sequence has one, a decode step. Rows from
cu[B] on (a batch padded to a fixed size) belong to no sequence and come out as zeros. 16-bit rows are
bfloat16 or float16. Index tensors are int32 on the cache's GPU; nothing here reads them on the host, so
every call can be captured into a graph. A page that a row needs but that is not in the cache (an entry
outside [0, pages), a position past the table's width) makes that row NaN, and a sequence whose ctx or start
is negative all of its rows; nothing else is touched. Nothing is recorded for autograd: a cache has no
gradient.

Everything runs on torch's current HIP stream; buffers are torch tensors on the caller's GPU. Arguments
of the usual form (dense, aligned) take a short way through native code; what follows it in each function
looks at every other form, copies what has to be dense, and refuses.
"""
from __future__ import annotations

import math

import torch

from . import _lib

F32 = torch.float32
PAGES = (16, 32, 64, 128)
HEAD_DIMS = (32, 64, 128)
_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_I32MAX = 2 ** 31 - 1


def _stream() -> int:
    return _lib.stream() if torch.cuda.is_initialized() else 0


def _require(ok, msg):
    if not ok:
        raise AssertionError(msg)


def new_cache(pages: int, Hkv: int, hd: int, page: int = 64, device="cuda"):
    """An empty cache of one layer: zero bytes, zero scales."""
    _require(page in PAGES, f"new_cache: page {page} not in {PAGES}")
    _require(hd in HEAD_DIMS, f"new_cache: head_dim {hd} not in {HEAD_DIMS}")
    _require(pages > 0 and Hkv > 0, f"new_cache: pages={pages} Hkv={Hkv}")
    z = lambda *shape, dt=torch.int8: torch.zeros(shape, dtype=dt, device=device)
    return z(pages, Hkv, page, hd), z(pages, Hkv, hd, page), z(pages, Hkv, dt=F32), z(pages, Hkv, dt=F32)


def _cache(fn, cache):
    """(k, v, ks, vs addresses, pages, page, Hkv, hd) of a checked cache."""
    k, v, ks, vs = cache
    n, Hkv, page, hd = k.shape
    if (k.dtype != torch.int8 or v.dtype != torch.int8 or v.shape != (n, Hkv, hd, page) or ks.dtype != F32 or vs.dtype != F32
            or ks.shape != (n, Hkv) or vs.shape != (n, Hkv)):
        raise AssertionError(f"{fn}: the cache is int8 k (pages, Hkv, page, hd) and v (pages, Hkv, hd, page), float32 ks and "
                             f"vs (pages, Hkv); got {[(tuple(x.shape), x.dtype) for x in cache]}")
    if not k.numel():
        raise AssertionError(f"{fn}: the cache is empty, k {tuple(k.shape)}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise AssertionError(f"{fn}: the cache's tensors must be contiguous")
    return k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), n, page, Hkv, hd


def _on_gpu(fn, dev):
    if dev.type != "cuda":
        raise AssertionError(f"{fn}: the cache must be on a GPU, got {dev}")


def _index(fn, name, x, n, dev):
    if x.dtype != torch.int32 or x.dim() != 1 or x.shape[0] != n or x.device != dev:
        raise AssertionError(f"{fn}: {name} must be int32 ({n},) on the cache's GPU, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x if x.is_contiguous() else x.contiguous()


def _table(fn, table, dev):
    if table.dtype != torch.int32 or table.dim() != 2 or table.device != dev:
        raise AssertionError(f"{fn}: the page table must be int32 (B, width) on the cache's GPU, got {table.dtype} "
                             f"{tuple(table.shape)} on {table.device}")
    if max(table.shape) > _I32MAX:
        raise AssertionError(f"{fn}: a page table of {tuple(table.shape)} entries, 2^31 or more on a side")
    return table if table.shape[1] < 2 or table.stride(1) == 1 else table.contiguous()


def _rows16(fn, name, x, dev):
    """A 16-bit tensor whose rows are dense and 16-byte aligned: x itself where it is so already."""
    if x.dtype not in _TYPES or x.device != dev:
        raise AssertionError(f"{fn}: {name} must be bfloat16 or float16 on the cache's GPU, got {x.dtype} on {x.device}")
    if x.shape[0] > _I32MAX:
        raise AssertionError(f"{fn}: {name} has {x.shape[0]} rows, 2^31 or more")
    dense = x.stride(-1) == 1 and (x.dim() == 2 or x.stride(1) == x.shape[2])
    return x if dense and x.stride(0) >= 0 and x.stride(0) % 8 == 0 and x.data_ptr() % 16 == 0 else x.clone(
        memory_format=torch.contiguous_format)


def _f32(fn, name, x, shape, dev):
    if x is None:
        return None
    if x.dtype != F32 or tuple(x.shape) != shape or x.device != dev:
        raise AssertionError(f"{fn}: {name} must be float32 {shape} on the cache's GPU, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x if x.is_contiguous() else x.contiguous()


def append(cache, qkv: torch.Tensor, table: torch.Tensor, ctx: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, cu=None,
           q_norm=None, k_norm=None, eps: float = 1e-6) -> torch.Tensor:
    """Put new tokens into the cache; returns their q heads (T, H, hd) for attend().

    qkv (T, (H + 2 Hkv) hd): q heads, k heads, v heads of every token. ctx (B,): tokens of each sequence
    that are cached already; the new ones follow. q and k heads are multiplied by w / sqrt(mean(x^2) + eps)
    where their weights q_norm, k_norm (fp32, hd) are given, then rotated with the rows of cos and sin (fp32,
    positions x hd) of their positions: x cos + (-hi, lo)(x) sin. A page's scale is max|x| / 127 over the
    tokens it holds; where new ones raise it, the older ones are rounded again. No two sequences' new
    tokens may share a page."""
    r = _lib.kv().append(*cache, qkv, table, ctx, cos, sin, cu, q_norm, k_norm, eps, _stream())
    if r is not None:
        return r if type(r) is not int else _lib.fail("uwc_kv_append", r)
    fn = "kv.append"
    k, v, ks, vs, pages, page, Hkv, hd = _cache(fn, cache)
    dev = cache[0].device
    _require(qkv.dim() == 2, f"{fn}: qkv must be (T, (H + 2 Hkv) hd), got {tuple(qkv.shape)}")
    T, wide = qkv.shape
    H = wide // hd - 2 * Hkv
    if wide % hd or H < 0:
        raise AssertionError(f"{fn}: qkv rows of {wide} do not hold 2 x {Hkv} kv heads of {hd} and whole q heads")
    table = _table(fn, table, dev)
    B, width = table.shape
    qkv = _rows16(fn, "qkv", qkv, dev)
    ctx = _index(fn, "ctx", ctx, B, dev)
    if cu is not None:
        cu = _index(fn, "cu", cu, B + 1, dev)
    elif T != B:
        raise AssertionError(f"{fn}: without cu every sequence has one row, got {T} rows for {B}")
    _require(cos.dim() == 2, f"{fn}: cos and sin must be (positions, {hd})")
    positions = cos.shape[0]
    cos, sin = _f32(fn, "cos", cos, (positions, hd), dev), _f32(fn, "sin", sin, (positions, hd), dev)
    q_norm, k_norm = _f32(fn, "q_norm", q_norm, (hd,), dev), _f32(fn, "k_norm", k_norm, (hd,), dev)
    _on_gpu(fn, dev)
    q = torch.empty((T, H, hd), dtype=qkv.dtype, device=dev)
    _lib.call("uwc_kv_append", qkv.data_ptr(), qkv.stride(0), _TYPES[qkv.dtype], T, B, None if cu is None else cu.data_ptr(),
              ctx.data_ptr(), table.data_ptr(), table.stride(0), width, cos.data_ptr(), sin.data_ptr(), positions,
              None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(), eps, H, Hkv, hd,
              page, pages, k, v, ks, vs, q.data_ptr(), _lib.stream())
    return q


def attend(cache, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, cu=None, max_new=None, max_len=None,
           window: int = 0, sinks: int = 0, scale=None) -> torch.Tensor:
    """Causal attention of new queries q (T, H, hd) over the cache: (T, H, hd) in q's type.

    lens (B,): tokens of each sequence in the cache, its new ones included; its queries are the last of
    them. H is a multiple of the cache's Hkv; q head i reads kv head i // (H / Hkv). window > 0: a query at
    position p sees keys above p - window, and the sequence's first `sinks`. Rows that see nothing are zeros.
    max_new, max_len: bounds of the sequences' new tokens and lengths that the caller knows, for splitting
    the work well; results are right for any. scale, above 0, defaults to 1 / sqrt(hd)."""
    r = _lib.kv().attend(*cache, q, table, lens, cu, max_new, max_len, window, sinks, scale, _stream())
    if r is not None:
        return r if type(r) is not int else _lib.fail("uwc_kv_attend", r)
    fn = "kv.attend"
    k, v, ks, vs, pages, page, Hkv, hd = _cache(fn, cache)
    dev = cache[0].device
    if q.dim() != 3 or q.shape[2] != hd or q.shape[1] < 1 or q.shape[1] % Hkv:
        raise AssertionError(f"{fn}: q must be (T, H, {hd}) with H a multiple of {Hkv}, got {tuple(q.shape)}")
    if window < 0 or sinks < 0 or (sinks and not window):
        raise AssertionError(f"{fn}: window={window} sinks={sinks} (sinks need a window)")
    T, H, _ = q.shape
    table = _table(fn, table, dev)
    B, width = table.shape
    q = _rows16(fn, "q", q, dev)
    lens = _index(fn, "lens", lens, B, dev)
    if cu is not None:
        cu = _index(fn, "cu", cu, B + 1, dev)
    elif T != B:
        raise AssertionError(f"{fn}: without cu every sequence has one row, got {T} rows for {B}")
    most = T if cu is not None else 1
    max_new = most if max_new is None else max(1, min(max_new, most))
    max_len = min(width * page if max_len is None else max(1, max_len), _I32MAX)
    window, sinks = min(window, _I32MAX), min(sinks, _I32MAX)
    _on_gpu(fn, dev)
    o = torch.empty((T, H, hd), dtype=q.dtype, device=dev)
    need = _lib.lib().uwc_kv_attend_scratch_bytes(T, B, int(cu is not None), H, Hkv, hd, max_new, max_len, window, sinks)
    scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib.call("uwc_kv_attend", k, v, ks, vs, pages, page, Hkv, hd, q.data_ptr(), q.stride(0), _TYPES[q.dtype], T, H,
              table.data_ptr(), table.stride(0), width, lens.data_ptr(), None if cu is None else cu.data_ptr(), B, max_new,
              max_len, window, sinks, 1.0 / math.sqrt(hd) if scale is None else scale,
              None if scratch is None else scratch.data_ptr(), need, o.data_ptr(), _lib.stream())
    return o


def read(cache, table: torch.Tensor, start: torch.Tensor, cu: torch.Tensor, rows: int, dtype=torch.bfloat16):
    """Cached tokens as values: keys and values (rows, Hkv, hd) of `dtype`, sequence b's tokens
    start[b] .. start[b] + cu[b + 1] - cu[b] - 1 at rows cu[b] .. cu[b + 1] - 1. rows is at least cu[B]."""
    if dtype in _TYPES:
        r = _lib.kv().read(*cache, table, start, cu, rows, _TYPES[dtype], _stream())
        if r is not None:
            return r if type(r) is not int else _lib.fail("uwc_kv_read", r)
    fn = "kv.read"
    k, v, ks, vs, pages, page, Hkv, hd = _cache(fn, cache)
    dev = cache[0].device
    _require(dtype in _TYPES, f"{fn}: dtype must be bfloat16 or float16, got {dtype}")
    _require(rows >= 0, f"{fn}: rows={rows}")
    table = _table(fn, table, dev)
    B, width = table.shape
    start, cu = _index(fn, "start", start, B, dev), _index(fn, "cu", cu, B + 1, dev)
    _on_gpu(fn, dev)
    ko = torch.empty((rows, Hkv, hd), dtype=dtype, device=dev)
    vo = torch.empty((rows, Hkv, hd), dtype=dtype, device=dev)
    _lib.call("uwc_kv_read", k, v, ks, vs, pages, page, Hkv, hd, table.data_ptr(), table.stride(0), width, start.data_ptr(),
              cu.data_ptr(), B, rows, _TYPES[dtype], ko.data_ptr(), vo.data_ptr(), _lib.stream())
    return ko, vo
