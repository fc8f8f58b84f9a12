"""Page operators of a KV cache, ``backend="hip"``: copies and compaction.

Both work on any cache tensor whose dimension ``page_dim`` numbers the pages
and whose trailing dimensions are one page's bytes: a layer's keys or values
(``page_dim=0``), or all planes and layers of a pool (``page_dim=2`` for
``[2, layers, pages, ...]``), 16-bit or packed.  One launch moves a page in
every plane.  ``PagePool.fork``, ``PagePool.make_writable`` and
``PagePool.compact`` say which pages to move.
"""

from __future__ import annotations

import torch

from . import hip_extension as ext


def _planes(cache, page_dim):
    """(planes, pages, bytes of a page in one plane)."""
    if type(page_dim) is not int or not 0 <= page_dim < cache.ndim:
        raise ValueError("page_dim must be a dimension of the cache")
    if not cache.is_contiguous() or cache.numel() == 0:
        raise ValueError("cache must be contiguous and not empty")
    planes = 1
    for size in cache.shape[:page_dim]:
        planes *= size
    pages = cache.shape[page_dim]
    return planes, pages, cache.numel() // (planes * pages) * cache.element_size()


def _check_moves(cache, pages, src_pages, dst_pages, backend, validate, rising):
    if backend != "hip":
        raise ValueError("page backend must be hip")
    for ids in (src_pages, dst_pages):
        if ids.ndim != 1 or ids.dtype != torch.int64 or not ids.is_contiguous():
            raise ValueError("source and destination pages must be contiguous int64 [moves]")
        if ids.device != cache.device:
            raise ValueError("page ids must share the cache device")
    if src_pages.numel() != dst_pages.numel():
        raise ValueError("source and destination pages must pair up")
    if src_pages.numel() > pages:
        raise ValueError("more moves than pages")
    if not validate:
        return
    src, dst = src_pages.tolist(), dst_pages.tolist()
    if any(page < 0 or page >= pages for page in (*src, *dst)):
        raise ValueError("physical block id out of range")
    if len(set(dst)) != len(dst):
        raise ValueError("a page cannot be the destination of two moves")
    if not set(src).isdisjoint(dst):
        raise ValueError("a page cannot be both source and destination")
    if rising and any(b <= a for a, b in zip(src, src[1:])):
        raise ValueError("source pages of a compaction must rise")
    if any(ext.share_bytes(cache, ids) for ids in (src_pages, dst_pages)):
        raise ValueError("page ids must not overlap the cache")


def _need_hip(cache):
    if cache.device.type != "cuda":
        raise ValueError("page operators require a HIP device")


def copy_kv_pages(cache, src_pages, dst_pages, *, page_dim=0, backend="hip", validate=True):
    """Page ``dst_pages[i]`` takes the content of page ``src_pages[i]``, in place, bit for bit.

    A source may feed several destinations.  ``validate=True`` reads the ids
    on the host and refuses pages out of range, a destination that occurs
    twice and a page that is both source and destination (the moves run at
    the same time); with ``validate=False`` moves with a page out of range are
    skipped, and the caller answers for the other two.
    """
    if backend == "hip" and not validate and ext.native.move_pages(cache, src_pages, dst_pages, None, page_dim):
        return
    planes, pages, page_bytes = _planes(cache, page_dim)
    _check_moves(cache, pages, src_pages, dst_pages, backend, validate, False)
    _need_hip(cache)
    if src_pages.numel() == 0:
        return
    lib = ext.load_hip_extension()
    with torch.cuda.device(cache.device):
        lib.call("mvme_copy_pages", cache.data_ptr(), planes, pages, page_bytes, src_pages.data_ptr(),
                 dst_pages.data_ptr(), src_pages.numel(), ext.current_stream(cache.device))


def compact_kv_pages(cache, src_pages, dst_pages, block_tables, *, page_dim=0, backend="hip", validate=True):
    """``copy_kv_pages``, and every entry of ``block_tables`` that is ``src_pages[i]`` becomes ``dst_pages[i]``.

    ``src_pages`` has to rise (``PagePool.compact`` returns them so).  Other
    entries, padding among them, stay.  block_tables: contiguous int64 of any
    shape, changed in place.
    """
    if (backend == "hip" and not validate and block_tables is not None
            and ext.native.move_pages(cache, src_pages, dst_pages, block_tables, page_dim)):
        return
    planes, pages, page_bytes = _planes(cache, page_dim)
    _check_moves(cache, pages, src_pages, dst_pages, backend, validate, True)
    if block_tables.dtype != torch.int64 or not block_tables.is_contiguous():
        raise ValueError("block tables must be a contiguous int64 tensor")
    if block_tables.device != cache.device:
        raise ValueError("block tables must share the cache device")
    if validate and any(ext.share_bytes(block_tables, t) for t in (cache, src_pages, dst_pages)):
        raise ValueError("block tables must not overlap the cache or the page ids")
    _need_hip(cache)
    if src_pages.numel() == 0:
        return
    lib = ext.load_hip_extension()
    with torch.cuda.device(cache.device):
        lib.call("mvme_compact_pages", cache.data_ptr(), planes, pages, page_bytes, src_pages.data_ptr(),
                 dst_pages.data_ptr(), src_pages.numel(), block_tables.data_ptr(), block_tables.numel(),
                 ext.current_stream(cache.device))
