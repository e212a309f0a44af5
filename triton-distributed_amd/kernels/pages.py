"""Pages of a paged KV cache: copy, reserve, fork, free, compact.

The reference has a dense cache only (``python/triton_dist/models/kv_cache.py:28-69``); what a server does with a paged
one between steps is here.  The state is three tensors on the GPU next to the pools:

* ``block_table`` int32 ``[B, max_pages]``: a row's pages from the front, -1 behind them;
* ``kv_lens`` int32 ``[B]``;
* ``page_refs`` int32 ``[pages]``: how many rows hold a page, 0 = free.

The pools are ``[pages, P, Hkv, D]``, or ``[layers, pages, P, Hkv, D]`` for all layers of a model at once (one table for
all of them).  Every function changes these tensors in place, enqueues its kernels through the C ABI in
``include/flash_decode.h`` (``fd_pages_*``) on the current (or given) stream and reads nothing on the host.  A free page is
handed out lowest id first, in the order of the requests.  Calls on one cache must follow each other on one stream.  ``stream=``
as in ``kernels/prefill.py``.
"""
from __future__ import annotations

from ctypes import byref
from typing import Optional, Union

import torch

from .._lib import FdPagePool, FdPageTables, load_library
from .flash_decode import _on
from .prefill import _check_devices, _check_int32, _launch, _need, _remember, _sig


def _pool(name, k_cache, v_cache) -> FdPagePool:
    """The pools' shape, checked; the addresses are the call's."""
    _need(k_cache.dim() in (4, 5) and v_cache.dim() == k_cache.dim() and k_cache.shape[:-2] == v_cache.shape[:-2],
          f"{name}: pools [pages, P, heads, dim] or [layers, pages, P, heads, dim] with the same pages")
    p = FdPagePool()
    p.layers = k_cache.shape[0] if k_cache.dim() == 5 else 1
    p.num_pages, p.page_size = k_cache.shape[-4], k_cache.shape[-3]
    for side, t in (("k", k_cache), ("v", v_cache)):
        rows, heads, dim = t.shape[-3:]
        _need(t.stride(-1) == 1 and (heads == 1 or t.stride(-2) == dim) and (rows == 1 or t.stride(-3) == heads * dim),
              f"{name}: a page must be contiguous")
        size = t.element_size()
        setattr(p, side + "_layer_stride", (t.stride(0) if t.dim() == 5 else 0) * size)
        # (a single page has no distance to a next one)
        setattr(p, side + "_page_stride", (t.stride(-4) if p.num_pages > 1 else rows * heads * dim) * size)
        setattr(p, side + "_page_bytes", rows * heads * dim * size)
    return p


def _tables(name, block_table, kv_lens, page_refs, num_pages) -> FdPageTables:
    _need(block_table.dim() == 2 and block_table.dtype == torch.int32
          and (block_table.shape[1] <= 1 or block_table.stride(1) == 1),
          f"{name}: block_table must be int32 [B, max_pages] with contiguous rows")
    _check_int32(name, "page_refs", page_refs, (num_pages,))
    t = FdPageTables()
    t.stride_table_bs = block_table.stride(0)
    t.batch, t.max_pages_per_seq = block_table.shape
    if kv_lens is not None:
        _check_int32(name, "kv_lens", kv_lens, (block_table.shape[0],))
    return t


_SEEN = {}   # pool and table images of calls whose arguments have been checked, by what the checks look at


def _checked(name, caches, tables, lists):
    """(fd_page_pool, fd_page_tables) of a call, checked once per kind of arguments.  caches: (k_cache, v_cache) or ();
    tables: (block_table, kv_lens or None, page_refs) or (); lists: further int32 tensors as (what, tensor, shape)."""
    key = (name, *map(_sig, caches), *map(_sig, tables), *((w, _sig(t), s) for w, t, s in lists))
    images = _SEEN.get(key)
    if images is None:
        _check_devices(name, *caches, *tables, *(t for _, t, _ in lists))
        pool = _pool(name, *caches) if caches else None
        for what, t, shape in lists:
            if t is not None:
                _check_int32(name, what, t, shape)
        pages = pool.num_pages if caches else tables[2].numel()
        images = _remember(_SEEN, key, (bytes(pool) if caches else None,
                                        bytes(_tables(name, *tables, pages)) if tables else None))
    pool = t = None
    if caches:
        pool = FdPagePool.from_buffer_copy(images[0])
        pool.k_cache, pool.v_cache = caches[0].data_ptr(), caches[1].data_ptr()
    if tables:
        t = FdPageTables.from_buffer_copy(images[1])
        t.block_table, t.page_refs = tables[0].data_ptr(), tables[2].data_ptr()
        if tables[1] is not None:
            t.kv_lens = tables[1].data_ptr()
    return pool, t


def paged_kv_copy(k_cache, v_cache, src_pages, dst_pages, *, stream=None):
    """Copies page ``src_pages[i]`` to page ``dst_pages[i]`` (int32 ``[n]``) in every layer of both pools.  The destinations
    must be distinct and none of them a source; ids outside the pool are skipped."""
    if stream is not None:
        return _on(stream, paged_kv_copy, k_cache, v_cache, src_pages, dst_pages)
    n = src_pages.numel()
    pool, _ = _checked("paged_kv_copy", (k_cache, v_cache), (), (("src_pages", src_pages, (n,)), ("dst_pages", dst_pages, (n,))))
    if n:
        _launch(load_library().fd_pages_copy, k_cache.device, byref(pool), src_pages.data_ptr(), dst_pages.data_ptr(), n)


def paged_kv_reserve(block_table, kv_lens, page_refs, new_tokens: Union[int, torch.Tensor], page_size: int, *,
                     ok_out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Gives every row the pages that its next ``new_tokens`` tokens need (an int for all rows, or int32 ``[B]``), so that
    the append that follows has somewhere to write.  Returns int32 ``[B]``: 1, or 0 where the table is too narrow, the pool has
    run out, or the row wants tokens but lacks a page for those that its length counts already (its length went up
    without pages: free it first) -- that row keeps what it had.  Rows are served in order; a row that gets nothing for want of
    free pages still counts against the rows behind it.  At most 4096 rows, and 2^20 new pages a row."""
    if stream is not None:
        return _on(stream, paged_kv_reserve, block_table, kv_lens, page_refs, new_tokens, page_size, ok_out=ok_out)
    each = new_tokens if isinstance(new_tokens, torch.Tensor) else None
    batch = block_table.shape[0]
    _, t = _checked("paged_kv_reserve", (), (block_table, kv_lens, page_refs),
                    (("new_tokens", each, (batch,)), ("ok_out", ok_out, (batch,))))
    if ok_out is None:
        ok_out = torch.empty(batch, dtype=torch.int32, device=block_table.device)
    _need(batch <= 4096, f"paged_kv_reserve: {batch} rows (at most 4096)")
    _need(each is not None or 0 <= new_tokens < 1 << 31, f"paged_kv_reserve: new_tokens {new_tokens}")
    if batch:
        _launch(load_library().fd_pages_reserve, block_table.device, byref(t), page_refs.numel(), int(page_size),
                each.data_ptr() if each is not None else None, 0 if each is not None else int(new_tokens), ok_out.data_ptr())
    return ok_out


def paged_kv_fork(k_cache, v_cache, block_table, kv_lens, page_refs, parents, children, *,
                  ok_out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Makes row ``children[i]`` a fork of row ``parents[i]`` (int32 ``[n]``): the parent's length, its full pages shared
    (counted, not copied), and of a part-filled last page a copy of its own, in every layer -- both rows can be appended to
    afterwards.  Returns int32 ``[n]``: 1, or 0 where a fork is refused and nothing changes (a row out of range or its own
    parent, a parent without a page for tokens that its length counts, a child that holds tokens or pages or was named
    before, no free page left).  Parents count as they are before
    the call.  At most 16384 forks."""
    if stream is not None:
        return _on(stream, paged_kv_fork, k_cache, v_cache, block_table, kv_lens, page_refs, parents, children, ok_out=ok_out)
    n = parents.numel()
    pool, t = _checked("paged_kv_fork", (k_cache, v_cache), (block_table, kv_lens, page_refs),
                       (("parents", parents, (n,)), ("children", children, (n,)), ("ok_out", ok_out, (n,))))
    if ok_out is None:
        ok_out = torch.empty(n, dtype=torch.int32, device=k_cache.device)
    if n:
        lib = load_library()
        need = lib.fd_pages_workspace_bytes(pool.num_pages, n)
        ws = torch.empty(need, dtype=torch.uint8, device=k_cache.device)
        _launch(lib.fd_pages_fork, k_cache.device, byref(pool), byref(t), parents.data_ptr(), children.data_ptr(), n,
                ok_out.data_ptr(), ws.data_ptr(), need)
    return ok_out


def paged_kv_free(block_table, kv_lens, page_refs, rows, *, stream=None):
    """Takes their pages from the listed rows (int32 ``[n]``): counts go down -- a page that no row holds any more is free --,
    the rows' entries become -1 and their lengths 0.  Empty rows, rows listed twice and rows out of range are skipped."""
    if stream is not None:
        return _on(stream, paged_kv_free, block_table, kv_lens, page_refs, rows)
    n = rows.numel()
    _, t = _checked("paged_kv_free", (), (block_table, kv_lens, page_refs), (("rows", rows, (n,)),))
    if n and t.batch:
        _launch(load_library().fd_pages_free, block_table.device, byref(t), page_refs.numel(), rows.data_ptr(), n)


def paged_kv_compact(k_cache, v_cache, block_table, page_refs, *, live_out: Optional[torch.Tensor] = None,
                     stream=None) -> torch.Tensor:
    """Moves the live pages to the front of the pool, in every layer: with ``n`` live pages, the k-th live page at or behind
    ``n`` goes to the k-th free page before ``n``; ``page_refs`` and ``block_table`` follow.  ``block_table`` must hold every
    row that holds pages; page ids kept anywhere else (a ``prefix_table`` that is no part of it) are not rewritten.  Returns
    int32 ``[1]`` (on the device): ``n``, from where on the pool is free."""
    if stream is not None:
        return _on(stream, paged_kv_compact, k_cache, v_cache, block_table, page_refs, live_out=live_out)
    pool, t = _checked("paged_kv_compact", (k_cache, v_cache), (block_table, None, page_refs), (("live_out", live_out, (1,)),))
    if live_out is None:
        live_out = torch.empty(1, dtype=torch.int32, device=k_cache.device)
    lib = load_library()
    need = lib.fd_pages_workspace_bytes(pool.num_pages, 0)
    ws = torch.empty(need, dtype=torch.uint8, device=k_cache.device)
    _launch(lib.fd_pages_compact, k_cache.device, byref(pool), byref(t), live_out.data_ptr(), ws.data_ptr(), need)
    return live_out
