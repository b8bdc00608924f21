"""Pages of the paged KV cache moved on the device, over the CUDA library.  No counterpart in the
reference, whose slots are ring buffers; the page lists come from ``g4b_b200.paging``
(``PagedKVManager.fork``, ``PagedKVManager.compact``)."""
from __future__ import annotations

import ctypes

from g4b_b200 import _cabi


def _pool(p, num_pages: int) -> tuple[int, int]:
    """Address and bytes of a page of one pool.  Only torch tensors come here (the pools of every layer, dozens in a call),
    so what is asked of a tensor is what costs least."""
    if not p.is_contiguous():
        raise ValueError("page pools must be contiguous")
    if p.dim() < 1 or p.shape[0] != num_pages:
        raise ValueError("page pools must all have the same number of pages (dim 0)")
    return p.data_ptr(), (p.nbytes // num_pages if num_pages else 0)


def copy_pages(pools, src_pages, dst_pages, *, stream=None):
    """``pool[dst_pages[i]] = pool[src_pages[i]]`` in every pool of ``pools``, in one launch
    (``g4b_page_copy``).  ``pools``: torch tensors ``[num_pages, ...]`` of any types, contiguous, with
    one number of pages: the K and V pools of all layers, and the scales of 8-bit ones.
    ``src_pages, dst_pages [n]`` int32 on the device; negative entries are padding.

    A page may be copied to many others.  A list that names one destination twice, or reads a
    page that it also writes, is not followed there (the entry is skipped and the device status
    word says so), so what it does never depends on the order of the blocks.  Returns None."""
    pools = list(pools)
    num_pages = int(pools[0].shape[0]) if pools and len(pools[0].shape) else 0
    a = _cabi.G4bPageCopyArgs()
    a.src_pages = _cabi.as_tensor(src_pages)
    a.dst_pages = _cabi.as_tensor(dst_pages)
    table = (_cabi.G4bPagePool * len(pools))()
    for p in pools:
        _cabi._check_device(p)
    flat = [x for p in pools for x in _pool(p, num_pages)]
    ctypes.memmove(table, (ctypes.c_int64 * len(flat))(*flat), 8 * len(flat))
    a.pools = table
    a.num_pages = num_pages
    a.num_pools = len(pools)
    _cabi.check(_cabi.load().g4b_page_copy(ctypes.byref(a), ctypes.c_void_p(_cabi.current_stream(stream))))
    return None
