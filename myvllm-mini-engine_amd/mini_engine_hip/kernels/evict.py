"""Eviction from a paged KV cache by attention weight, ``backend="hip"``.

Of a sequence that has grown past its bound, each layer and kv head keeps its
first tokens, its most recent ones and those of the others that received most
attention (``kernels/weights.py`` keeps the account); their rows move to the
front of the sequence's pages.  Keys are cached rotated, so they may stand
anywhere.  ``PagePool.truncate`` gives back the pages behind them, and
``KVCachePool.evict`` runs all layers of a pool.
"""

from __future__ import annotations

import torch

from . import hip_extension as ext
from .paged import MAX_TABLE_CAPACITY
from .shared import check_aligned
from .weights import check_weights


def _check_pages(tables, lengths, firsts, block_size, num_blocks, keep):
    """Host-synchronising checks of the metadata."""
    writers = {}
    for b, (table, n, first) in enumerate(zip(tables, lengths, firsts)):
        if not 0 < n <= len(table) * block_size:
            raise ValueError("invalid context length")
        if any(page < 0 or page >= num_blocks for page in table[:-(-n // block_size)]):
            raise ValueError("physical block id out of range")
        if first < 0:
            raise ValueError("first must not be negative")
        if n > keep:
            for page in table[min(first, keep) // block_size:-(-keep // block_size)]:
                writers.setdefault(page, []).append(b)
    readers = [(page, b) for b, (table, n) in enumerate(zip(tables, lengths)) for page in table[:-(-n // block_size)]]
    for page, b in readers:
        if any(other != b for other in writers.get(page, ())):
            raise ValueError("eviction would write into a page that another sequence holds")
    for b, (table, n) in enumerate(zip(tables, lengths)):
        used = table[:-(-n // block_size)]
        if n > keep and len(set(used)) != len(used):
            raise ValueError("a sequence names a page twice")


def evict_kv_cache(key_cache, value_cache, weights, block_tables, context_lens, block_size, keep, *, first=None,
                   recent=0, backend="hip", validate=True):
    """Keep ``keep`` tokens of every sequence that has more, per layer and kv head.

    key_cache/value_cache [num_blocks, block_size, Hkv, D], or all layers
    [layers, num_blocks, block_size, Hkv, D] with weights [layers, B, Hkv, S]
    (one layer: [B, Hkv, S]), S at least the tables' capacity.  Always kept are
    a sequence's ``first[b]`` leading tokens (int64 [B]; None: none) and its
    ``recent`` last ones, as far as ``keep`` reaches; of those between the ones
    with the largest weights (NaN above every number, ties to the lowest
    position).  Their rows move to positions ``0 .. keep - 1``, in order, in
    place; what lies behind stays as it was.

    Returns (kept, lengths, weights), new tensors: the position that each row
    came from, int64 [(layers,) B, Hkv, min(keep, S)] with -1 behind the last;
    the new context lengths; the kept tokens' weights, zero behind the last.

    ``validate=True`` reads the metadata on the host and refuses lengths and
    pages that cannot be, and rows that would move into a page that another
    sequence of the batch holds too (protect shared prefixes with ``first``, or
    ``PagePool.make_writable`` them).  With ``validate=False`` (graph capture)
    the caller answers for that; a sequence whose length cannot be (0: an empty
    row of a padded batch) keeps its length and its rows, and its line of the new
    weights is zero (``weights`` itself never changes).
    """
    if backend != "hip":
        raise ValueError("eviction backend must be hip")
    if not validate:
        result = ext.native.evict(key_cache, value_cache, weights, block_tables, context_lens, block_size, keep, first,
                                  recent)
        if result is not None:
            return result
    if (key_cache.ndim not in (4, 5) or value_cache.shape != key_cache.shape or any(size <= 0 for size in key_cache.shape)
            or not key_cache.is_contiguous() or not value_cache.is_contiguous()):
        raise ValueError("KV caches must be contiguous [(layers,) pages, block_size, kv_heads, head_dim]")
    if key_cache.dtype not in (torch.float16, torch.bfloat16) or value_cache.dtype != key_cache.dtype:
        raise ValueError("KV cache requires FP16/BF16")
    layers = key_cache.shape[0] if key_cache.ndim == 5 else 1
    num_blocks, size, kv_heads, head_dim = key_cache.shape[-4:]
    if size != block_size:
        raise ValueError("block size mismatch")
    if head_dim % 8 or head_dim > 1024:
        raise ValueError("eviction requires head_dim a multiple of 8 up to 1024")
    if (block_tables.ndim != 2 or block_tables.shape[0] <= 0 or block_tables.shape[1] <= 0 or context_lens.ndim != 1
            or context_lens.shape[0] != block_tables.shape[0]):
        raise ValueError("block tables and context lengths do not match the batch")
    batch, width = block_tables.shape
    metadata = [block_tables, context_lens]
    if first is not None:
        if first.ndim != 1 or first.shape[0] != batch:
            raise ValueError("first must be [sequences]")
        metadata.append(first)
    if any(t.dtype != torch.int64 or not t.is_contiguous() for t in metadata):
        raise ValueError("block tables, context lengths and first must be contiguous int64 tensors")
    if width * block_size > MAX_TABLE_CAPACITY:
        raise ValueError("maximum table capacity is 1M tokens")
    if type(keep) is not int or keep <= 0 or type(recent) is not int or recent < 0:
        raise ValueError("keep must be a positive integer and recent a nonnegative one")
    if any(t.device != key_cache.device for t in (value_cache, *metadata)):
        raise ValueError("caches and metadata must share a device")
    lines = (layers, batch, kv_heads) if key_cache.ndim == 5 else (batch, kv_heads)
    check_weights(weights, lines, width * block_size, key_cache.device)
    inputs = (weights, *metadata)
    if (ext.share_bytes(key_cache, value_cache)
            or any(ext.share_bytes(cache, t) for cache in (key_cache, value_cache) for t in inputs)):
        raise ValueError("caches must not overlap each other or the inputs")
    if validate:
        firsts = [0] * batch if first is None else first.tolist()
        _check_pages(block_tables.tolist(), context_lens.tolist(), firsts, block_size, num_blocks, keep)
    if key_cache.device.type != "cuda":
        raise ValueError("eviction requires a HIP device")
    check_aligned(key_cache, value_cache)
    lib = ext.load_hip_extension()
    row = weights.shape[-1]
    with torch.cuda.device(key_cache.device):
        kept = torch.empty((*lines, min(keep, row)), dtype=torch.int64, device=key_cache.device)
        lengths = torch.empty_like(context_lens)
        new_weights = torch.empty_like(weights)
        lib.call("mvme_evict_kv_cache", key_cache.data_ptr(), value_cache.data_ptr(), weights.data_ptr(),
                 new_weights.data_ptr(), row, kept.data_ptr(), lengths.data_ptr(), block_tables.data_ptr(),
                 context_lens.data_ptr(), first.data_ptr() if first is not None else None, layers, batch, kv_heads,
                 head_dim, num_blocks, block_size, width, min(keep, row), min(recent, row), ext.dtype_code(key_cache.dtype),
                 ext.current_stream(key_cache.device))
    return kept, lengths, new_weights
