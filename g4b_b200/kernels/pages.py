"""Pages of the paged KV cache moved on the device, over the CUDA library.  No counterpart in the
reference, whose slots are ring buffers; the page lists come from ``g4b_b200.paging``
(``PagedKVManager.fork``, ``PagedKVManager.compact``)."""
from __future__ import annotations

import ctypes
import struct

from g4b_b200 import _cabi

_HEAD, _TAIL = struct.Struct("@Pq"), struct.Struct("@ii")      # G4bPageCopyArgs around its two views


def copy_pages(pools, src_pages, dst_pages, *, stream=None):
    """``pool[dst_pages[i]] = pool[src_pages[i]]`` in every pool of ``pools``, in one launch
    (``g4b_page_copy``).  ``pools``: torch tensors ``[num_pages, ...]`` of any types, contiguous, with
    one number of pages: the K and V pools of all layers, and the scales of 8-bit ones.
    ``src_pages, dst_pages [n]`` int32 on the device, n at most 65536; negative entries are padding.

    A page may be copied to many others.  A list that names one destination twice, or reads a
    page that it also writes, is not followed there (the entry is skipped and the device status
    word says so), so what it does never depends on the order of the blocks; lists handed out by several
    calls of the manager go through ``g4b_b200.paging.copy_stages`` first.  Returns None."""
    pools = list(pools)
    if _cabi.page_copy(pools, src_pages, dst_pages, stream):
        return None
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
    if num_pages:
        flat[1::2] = [p.nbytes // num_pages for p in pools]
    a = _cabi.G4bPageCopyArgs.from_buffer_copy(
        _HEAD.pack(0, num_pages) + _cabi.views(src_pages, dst_pages) + _TAIL.pack(len(pools), 0))
    table = struct.pack(f"@{len(flat)}q", *flat)
    a.pools = ctypes.cast(ctypes.c_char_p(table), ctypes.POINTER(_cabi.G4bPagePool))
    _cabi.check(_cabi.load().g4b_page_copy(ctypes.byref(a), _cabi.current_stream(stream)))
    return None
