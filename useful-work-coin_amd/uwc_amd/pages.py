"""Which page of the paged 8-bit cache (uwc_amd.kv) belongs to whom, on MI355X: sequences that branch (samples of one
prompt, beams), end and grow share pages, copy the one they still write, and give back what nobody holds; a pool with
holes is moved together. No counterpart in the reference, whose DetQwen3.generate_greedy keeps whole rows of one
sequence (runtime/detrt/qwen3.py:296-334).

Every layer's cache has the same pages, and the page table (int32 (B, width)) names a sequence's pages in all of them; entries
past a sequence's pages are -1. refs (int32 (pages,)) counts who holds a page: rows of the table, and others that the
caller adds, as for a prompt's pages kept for later. A page with no holder is free.

  fork      the table's rows become copies of others: branch, reorder, end (parent -1) and grow in one call
  compact   the pages in use move to the front of the pool
  new_refs  counts of a pool that nobody holds anything of

Tables, lengths and counts come out as new tensors, the caches change in place. Index tensors are int32 on the cache's GPU;
nothing here reads them on the host, so every call can be captured into a graph. Entries of a table outside
[0, pages) are pages that are not there, kept as they are. Counts have to be right: a page that two rows name with a count
of one may be handed out while the second still reads it (nothing outside the pool is ever touched).

Everything runs on torch's current HIP stream; buffers are torch tensors on the caller's GPU. Arguments of the usual form
take the short way of uwc_amd.kv.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, kv

ROWS = 4096
_I32MAX = 2 ** 31 - 1


def new_refs(pages: int, device="cuda") -> torch.Tensor:
    """Counts of a pool of free pages."""
    return torch.zeros(pages, dtype=torch.int32, device=device)


def _checked(fn, caches, table, refs):
    """(pointers, pages, page, Hkv, hd, table) of checked arguments."""
    if not caches:
        raise AssertionError(f"{fn}: no caches")
    shape, dev = caches[0][0].shape, caches[0][0].device
    ptrs = []
    for c in caches:
        k, v, ks, vs, pages, page, Hkv, hd = kv._cache(fn, c)
        if c[0].shape != shape or any(x.device != dev for x in c):
            raise AssertionError(f"{fn}: all layers' caches must be of one shape on one GPU, got k {tuple(c[0].shape)} on {c[0].device} "
                                 f"beside {tuple(shape)} on {dev}")
        ptrs += [k, v, ks, vs]
    table = kv._table(fn, table, dev)
    if table.shape[0] > ROWS:
        raise AssertionError(f"{fn}: a table of {table.shape[0]} rows, more than {ROWS}")
    refs = kv._index(fn, "refs", refs, pages, dev)
    kv._on_gpu(fn, dev)
    return (ctypes.c_void_p * len(ptrs))(*ptrs), pages, page, Hkv, hd, table, refs


def fork(caches, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor, room: int = 0):
    """(table, lens, refs, missing): row i of the new table continues old row parents[i], which has lens[parents[i]] tokens.

    caches: every layer's (k, v, ks, vs). parents (R,) int32: -1 (or any number that is no row) leaves a row empty, of length 0; old rows
    that are nobody's parent let their pages go. The first row of a parent keeps its pages; the others share the
    full ones and get a copy of the last, partly filled one (of its first tokens, up to a multiple of 16, in every layer; what
    lies behind them is not defined), as does the first where refs says that others hold that page too. Then every row
    gets pages for `room` more tokens, as far as the table is wide. Pages are the lowest free ones, in the order of rows and
    entries; where there are too few, entries stay -1 and missing (1,) int32 counts them."""
    r = _lib.kv().fork(caches, table, lens, refs, parents, room, kv._stream())
    if r is not None:
        return r if type(r) is not int else _lib.fail("uwc_kv_fork", r)
    fn = "pages.fork"
    if room < 0:
        raise AssertionError(f"{fn}: room={room}")
    ptrs, pages, page, Hkv, hd, table, refs = _checked(fn, caches, table, refs)
    dev = refs.device
    B, width = table.shape
    lens = kv._index(fn, "lens", lens, B, dev)
    R = parents.shape[0] if parents.dim() == 1 else -1
    parents = kv._index(fn, "parents", parents, R, dev)
    if R > ROWS:
        raise AssertionError(f"{fn}: {R} parents, more than {ROWS}")
    with torch.cuda.device(dev):
        new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=dev)  # noqa: E731
        table_, lens_, refs_, missing = new(R, width), new(R), new(pages), new(1)
        need = _lib.lib().uwc_kv_pages_scratch_bytes(pages, R)
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.call("uwc_kv_fork", len(caches), ptrs, pages, page, Hkv, hd, table.data_ptr(), table.stride(0), width, lens.data_ptr(), B,
                  refs.data_ptr(), parents.data_ptr(), R, min(room, _I32MAX), table_.data_ptr(), lens_.data_ptr(), refs_.data_ptr(),
                  missing.data_ptr(), scratch.data_ptr(), need, _lib.stream())
    return table_, lens_, refs_, missing


def compact(caches, table: torch.Tensor, refs: torch.Tensor):
    """(table, refs) after the pages in use, n of them, have moved to the first n places of the pool, in every layer: those
    from n on, in their order, to the free ones before n; the others stay. A pool may then be cut to its first n pages.

    All pages in use move, but only the table is renamed: who holds pages without being a row of it gives them as a row of this
    call, of their numbers alone, and reads the new ones there."""
    r = _lib.kv().compact(caches, table, refs, kv._stream())
    if r is not None:
        return r if type(r) is not int else _lib.fail("uwc_kv_compact", r)
    fn = "pages.compact"
    ptrs, pages, page, Hkv, hd, table, refs = _checked(fn, caches, table, refs)
    dev = refs.device
    B, width = table.shape
    with torch.cuda.device(dev):
        table_ = torch.empty((B, width), dtype=torch.int32, device=dev)
        refs_ = torch.empty(pages, dtype=torch.int32, device=dev)
        need = _lib.lib().uwc_kv_pages_scratch_bytes(pages, 0)
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.call("uwc_kv_compact", len(caches), ptrs, pages, page, Hkv, hd, table.data_ptr(), table.stride(0), width, B,
                  refs.data_ptr(), table_.data_ptr(), refs_.data_ptr(), scratch.data_ptr(), need, _lib.stream())
    return table_, refs_
