"""Pages of the paged KV cache moved on the device, over the CUDA library.  No counterpart in the
reference, whose slots are ring buffers; the page lists come from ``g4b_b200.paging``
(``PagedKVManager.fork``, ``PagedKVManager.compact``)."""
from __future__ import annotations

import ctypes
import struct

from g4b_b200 import _cabi


def copy_pages(pools, src_pages, dst_pages, *, stream=None):
    """``pool[dst_pages[i]] = pool[src_pages[i]]`` in every pool of ``pools``, in one launch
    (``g4b_page_copy``).  ``pools``: torch tensors ``[num_pages, ...]`` of any types, contiguous, with
    one number of pages: the K and V pools of all layers, and the scales of 8-bit ones.
    ``src_pages, dst_pages [n]`` int32 on the device; negative entries are padding.

    A page may be copied to many others.  A list that names one destination twice, or reads a
    page that it also writes, is not followed there (the entry is skipped and the device status
    word says so), so what it does never depends on the order of the blocks.  Returns None."""
    # (the pools are dozens: what is asked of each is what costs least)
    pools = list(pools)
    shapes = [p.shape for p in pools]
    num_pages = shapes[0][0] if pools and shapes[0] else 0
    for device in {p.get_device() for p in pools}:
        _cabi._check_device(next(p for p in pools if p.get_device() == device))
    if not all([p.is_contiguous() for p in pools]):
        raise ValueError("page pools must be contiguous")
    if [s for s in shapes if not s or s[0] != num_pages]:
        raise ValueError("page pools must all have the same number of pages (dim 0)")
    flat = [0] * (2 * len(pools))
    flat[::2] = [p.data_ptr() for p in pools]
    flat[1::2] = [p.nbytes for p in pools] if num_pages < 2 else [p.nbytes // num_pages for p in pools]
    table = (_cabi.G4bPagePool * len(pools)).from_buffer_copy(struct.pack(f"@{len(flat)}q", *flat))
    a = _cabi.G4bPageCopyArgs(table, num_pages)
    a.src_pages = _cabi.as_tensor(src_pages)
    a.dst_pages = _cabi.as_tensor(dst_pages)
    a.num_pools = len(pools)
    _cabi.check(_cabi.load().g4b_page_copy(ctypes.byref(a), ctypes.c_void_p(_cabi.current_stream(stream))))
    return None
