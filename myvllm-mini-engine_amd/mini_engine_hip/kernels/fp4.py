"""The KV cache in 4 bits, ``backend="hip"``: writing, reading back, attention.

Counterparts of the 16-bit entry points (``data.py``, ``paged.py``,
``prefill.py``) with their metadata, validation and error conventions, over a
packed cache: uint8 ``[pages, kv_heads, record]``, one record per page and kv
head.  A record (``fp4_record_bytes``) holds ``block_size`` tokens: their E2M1
codes, token-major, ``head_dim / 2`` bytes each with the even dim in the low
four bits, then one E8M0 scale byte per 32 dims, then padding to 16 bytes.
``include/mvme_fp4.h`` has the rounding rule.  17 bytes hold what takes 64 in
16 bits; every stored value is exact in fp16 and in bf16.

Rows come in rotated, as the 16-bit cache takes them: ``qk_norm_rope_write_kv``
into a 16-bit staging page and ``write_kv_cache_slots_fp4`` from there.
"""

from __future__ import annotations

import torch

from . import hip_extension as ext
from .data import _row_stride

HEAD_DIMS = (32, 64, 96, 128, 192, 256)  # attention; writing and reading take every multiple of 32 up to 256
MAX_TABLE_CAPACITY = 1048576
_HALF = (torch.float16, torch.bfloat16)


def _check(condition, message):
    if not condition:
        raise RuntimeError(message)


def _backend(backend, what):
    if backend != "hip":
        raise ValueError(f"packed {what} backend must be hip")


def fp4_record_bytes(block_size, head_dim):
    """Bytes of one record of a packed cache: ``block_size`` tokens of one kv head."""
    if type(block_size) is not int or not 0 < block_size <= MAX_TABLE_CAPACITY:
        raise ValueError("block_size must be a positive integer of at most 1M tokens")
    if type(head_dim) is not int or head_dim <= 0 or head_dim > 256 or head_dim % 32:
        raise ValueError("packed KV cache requires head_dim a multiple of 32 up to 256")
    return -(-block_size * (head_dim // 2 + head_dim // 32) // 16) * 16


def _check_caches(key_cache, value_cache, block_size, head_dim):
    record = fp4_record_bytes(block_size, head_dim)
    if (key_cache.ndim != 3 or value_cache.shape != key_cache.shape or key_cache.shape[2] != record
            or any(size <= 0 for size in key_cache.shape)
            or key_cache.dtype != torch.uint8 or value_cache.dtype != torch.uint8
            or not key_cache.is_contiguous() or not value_cache.is_contiguous()):
        raise ValueError("packed KV caches must be contiguous uint8 [pages, kv_heads, fp4_record_bytes]")
    if any(t.device.type == "cuda" and t.data_ptr() % 16 for t in (key_cache, value_cache)):
        raise ValueError("packed KV caches must be 16-byte aligned")


def _check_rows(key_cache, key, value):
    if key.ndim != 3 or value.shape != key.shape or key.shape[1] != key_cache.shape[1]:
        raise ValueError("packed key/value must be [tokens, kv_heads, head_dim] matching the cache")
    if key.dtype not in _HALF or value.dtype != key.dtype:
        raise ValueError("packed KV rows require FP16/BF16")


def _check_devices(first, others):
    for tensor in others:
        if tensor.device != first.device:
            raise ValueError("packed KV tensors must share the cache device")


def _need_hip(tensor):
    if tensor.device.type != "cuda":
        raise ValueError("packed KV caches require a HIP device")


def write_kv_cache_slots_fp4(key_cache, value_cache, slot_mapping, key, value, block_size, *, backend="hip",
                             validate=True):
    """Quantise row t of ``key``/``value`` into cache slot ``slot_mapping[t]``.

    A slot is ``page * block_size + offset``.  As with ``write_kv_cache_slots``,
    ``validate=True`` reads the slots on the host, which must be in range and
    distinct, and refuses sources that alias a cache; with ``validate=False``
    (graph capture) the kernel skips slots outside the pool.  The sources may
    be strided views whose per-token ``[kv_heads, head_dim]`` rows are dense.
    """
    _backend(backend, "data")
    if not validate and ext.native.fp4_write_slots(key_cache, value_cache, slot_mapping, key, value, block_size):
        return
    if key.ndim != 3:
        raise ValueError("packed key/value must be [tokens, kv_heads, head_dim] matching the cache")
    tokens, _, head_dim = key.shape
    _check_caches(key_cache, value_cache, block_size, head_dim)
    _check_rows(key_cache, key, value)
    if (slot_mapping.ndim != 1 or slot_mapping.numel() != tokens or slot_mapping.dtype != torch.int64
            or not slot_mapping.is_contiguous()):
        raise ValueError("slot_mapping must be contiguous int64 [tokens]")
    _check_devices(key_cache, (value_cache, slot_mapping, key, value))
    if validate:
        slots = slot_mapping.tolist()
        capacity = key_cache.shape[0] * block_size
        if any(slot < 0 or slot >= capacity for slot in slots):
            raise ValueError("KV slot is outside cache capacity")
        if len(set(slots)) != len(slots):
            raise ValueError("duplicate KV slots would race during scatter")
        _refuse_aliases(key_cache, value_cache, (key, value, slot_mapping))
    _need_hip(key_cache)
    if tokens == 0:
        return
    key_stride, key = _row_stride(key)
    value_stride, value = _row_stride(value)
    lib = ext.load_hip_extension()
    with torch.cuda.device(key_cache.device):
        lib.call("mvme_fp4_write_slots", key_cache.data_ptr(), value_cache.data_ptr(), key_cache.shape[0], block_size,
                 key_cache.shape[1], head_dim, slot_mapping.data_ptr(), key.data_ptr(), value.data_ptr(), tokens,
                 key_stride, value_stride, ext.dtype_code(key.dtype), ext.current_stream(key_cache.device))


def _refuse_aliases(key_cache, value_cache, sources):
    if (ext.share_bytes(key_cache, value_cache)
            or any(ext.share_bytes(cache, source) for cache in (key_cache, value_cache) for source in sources)):
        raise ValueError("KV destinations and source tensors must not overlap")


def write_kv_cache_batch_fp4(key_cache, value_cache, block_tables, token_offsets, key, value, block_size, *,
                             backend="hip", validate=True):
    """Decode-step write: row b goes to position ``token_offsets[b]`` of the pages ``block_tables[b]``."""
    _backend(backend, "data")
    if not validate and ext.native.fp4_write_batch(key_cache, value_cache, block_tables, token_offsets, key, value,
                                                   block_size):
        return
    if key.ndim != 3:
        raise ValueError("packed key/value must be [tokens, kv_heads, head_dim] matching the cache")
    batch, _, head_dim = key.shape
    _check_caches(key_cache, value_cache, block_size, head_dim)
    _check_rows(key_cache, key, value)
    if (block_tables.ndim != 2 or token_offsets.ndim != 1 or block_tables.shape[0] != batch
            or token_offsets.shape[0] != batch or block_tables.shape[1] <= 0):
        raise ValueError("batch block table or offset shape mismatch")
    if any(t.dtype != torch.int64 or not t.is_contiguous() for t in (block_tables, token_offsets)):
        raise ValueError("batch block tables and offsets must be contiguous int64 tensors")
    _check_devices(key_cache, (value_cache, block_tables, token_offsets, key, value))
    if validate:
        positions, tables = token_offsets.tolist(), block_tables.tolist()
        slots = set()
        for position, table in zip(positions, tables):
            if not 0 <= position < len(table) * block_size:
                raise ValueError("batch KV offset out of range")
            page = table[position // block_size]
            if not 0 <= page < key_cache.shape[0]:
                raise ValueError("KV batch physical block id out of range")
            slots.add(page * block_size + position % block_size)
        if len(slots) != batch:
            raise ValueError("duplicate KV slots would race during scatter")
        _refuse_aliases(key_cache, value_cache, (key, value, block_tables, token_offsets))
    _need_hip(key_cache)
    if batch == 0:
        return
    key_stride, key = _row_stride(key)
    value_stride, value = _row_stride(value)
    lib = ext.load_hip_extension()
    with torch.cuda.device(key_cache.device):
        lib.call("mvme_fp4_write_batch", key_cache.data_ptr(), value_cache.data_ptr(), key_cache.shape[0], block_size,
                 key_cache.shape[1], head_dim, block_tables.data_ptr(), block_tables.shape[1],
                 token_offsets.data_ptr(), key.data_ptr(), value.data_ptr(), batch, key_stride, value_stride,
                 ext.dtype_code(key.dtype), ext.current_stream(key_cache.device))


def gather_kv_cache_slots_fp4(key_cache, value_cache, slot_mapping, block_size, head_dim, dtype, *, backend="hip",
                              validate=True):
    """K and V rows ``[tokens, kv_heads, head_dim]`` of the slots, in 16 bits (exact).

    ``validate=False`` reads slots outside the pool as zeros.
    """
    _backend(backend, "data")
    if not validate:
        rows = ext.native.fp4_gather_slots(key_cache, value_cache, slot_mapping, block_size, head_dim, dtype)
        if rows is not None:
            return rows
    _check_caches(key_cache, value_cache, block_size, head_dim)
    if dtype not in _HALF:
        raise ValueError("packed KV rows require FP16/BF16")
    if slot_mapping.ndim != 1 or slot_mapping.dtype != torch.int64 or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous int64 [tokens]")
    _check_devices(key_cache, (value_cache, slot_mapping))
    if validate:
        capacity = key_cache.shape[0] * block_size
        if any(slot < 0 or slot >= capacity for slot in slot_mapping.tolist()):
            raise ValueError("KV slot is outside cache capacity")
    _need_hip(key_cache)
    tokens, kv_heads = slot_mapping.numel(), key_cache.shape[1]
    rows = torch.empty((2, tokens, kv_heads, head_dim), dtype=dtype, device=key_cache.device)
    if tokens:
        lib = ext.load_hip_extension()
        with torch.cuda.device(key_cache.device):
            lib.call("mvme_fp4_gather_slots", rows[0].data_ptr(), rows[1].data_ptr(), key_cache.data_ptr(),
                     value_cache.data_ptr(), key_cache.shape[0], block_size, kv_heads, head_dim,
                     slot_mapping.data_ptr(), tokens, ext.dtype_code(dtype), ext.current_stream(key_cache.device))
    return rows[0], rows[1]


def gather_kv_cache_fp4(key_cache, value_cache, block_ids, token_count, block_size, head_dim, dtype, *, backend="hip",
                        validate=True):
    """K and V rows of positions ``[0, token_count)`` of a page list, in 16 bits (exact).

    ``validate=False`` reads pages outside the pool as zeros.
    """
    _backend(backend, "data")
    _check_caches(key_cache, value_cache, block_size, head_dim)
    if dtype not in _HALF:
        raise ValueError("packed KV rows require FP16/BF16")
    if block_ids.ndim != 1 or block_ids.dtype != torch.int64 or not block_ids.is_contiguous():
        raise ValueError("block_ids must be contiguous int64 [pages]")
    if token_count < 0:
        raise ValueError("token_count cannot be negative")
    if token_count > block_ids.numel() * block_size:
        raise ValueError("token_count exceeds supplied block table capacity")
    _check_devices(key_cache, (value_cache, block_ids))
    if validate and any(page < 0 or page >= key_cache.shape[0] for page in block_ids.tolist()):
        raise ValueError("KV physical block id out of range")
    _need_hip(key_cache)
    kv_heads = key_cache.shape[1]
    rows = torch.empty((2, token_count, kv_heads, head_dim), dtype=dtype, device=key_cache.device)
    if token_count:
        lib = ext.load_hip_extension()
        with torch.cuda.device(key_cache.device):
            lib.call("mvme_fp4_gather", rows[0].data_ptr(), rows[1].data_ptr(), key_cache.data_ptr(),
                     value_cache.data_ptr(), key_cache.shape[0], block_size, kv_heads, head_dim,
                     block_ids.data_ptr(), block_ids.numel(), token_count, ext.dtype_code(dtype),
                     ext.current_stream(key_cache.device))
    return rows[0], rows[1]


def fp4_workspace_bytes(batch, q_heads, kv_heads, head_dim, block_size, table_width, partition_tokens=0):
    """Bytes of the partition workspace paged_attention_fp4 needs for these shapes (0: none)."""
    return ext.load_hip_extension().fp4_workspace_size(batch, q_heads, kv_heads, head_dim, block_size, table_width,
                                                       partition_tokens)


def paged_attention_fp4(query, key_cache, value_cache, block_tables, context_lens, block_size, *, backend="hip",
                        validate=True, partition_tokens=0, out=None, workspace=None):
    """Decode attention over a packed KV cache: ``paged_attention`` on 4-bit pages.

    query [B, Hq, D] fp16/bf16, block_tables [B, W] and context_lens [B] int64;
    returns [B, Hq, D] in the query's type.  ``validate=False`` reads no
    metadata on the host (graph capture); sequences whose length is not
    positive or passes the table give zeros and pages out of range are
    skipped.  A NaN block of a value reaches its own 32 dims of the output.
    ``partition_tokens`` (0 = library plan) splits sequences over
    work-groups; ``out`` / ``workspace`` may supply the buffers.
    """
    _backend(backend, "decode")
    if not validate and out is None and workspace is None:
        result = ext.native.fp4_decode(query, key_cache, value_cache, block_tables, context_lens, block_size,
                                       partition_tokens)
        if result is not None:
            return result
    if query.dtype not in _HALF:
        raise ValueError("HIP paged attention supports FP16/BF16")
    if query.ndim != 3 or any(size <= 0 for size in query.shape):
        raise ValueError("query must be [batch, q_heads, head_dim], not empty")
    batch, q_heads, head_dim = query.shape
    if head_dim not in HEAD_DIMS:
        raise ValueError("packed attention supports head_dim 32,64,96,128,192,256")
    _check_caches(key_cache, value_cache, block_size, head_dim)
    num_blocks, kv_heads, _ = key_cache.shape
    if q_heads % kv_heads:
        raise ValueError("query heads must be divisible by the cache's kv heads")
    if (block_tables.ndim != 2 or block_tables.shape[0] != batch or block_tables.shape[1] <= 0
            or context_lens.ndim != 1 or context_lens.shape[0] != batch):
        raise ValueError("block tables and context lengths do not match the batch")
    if any(t.dtype != torch.int64 or not t.is_contiguous() for t in (block_tables, context_lens)):
        raise ValueError("block tables and context lengths must be contiguous int64 tensors")
    width = block_tables.shape[1]
    if width * block_size > MAX_TABLE_CAPACITY:
        raise ValueError("maximum table capacity is 1M tokens")
    if type(partition_tokens) is not int or partition_tokens < 0:
        raise ValueError("partition_tokens must be a nonnegative integer")
    _check_devices(query, (key_cache, value_cache, block_tables, context_lens))
    if out is not None and (out.shape != query.shape or out.dtype != query.dtype or out.device != query.device
                            or not out.is_contiguous()):
        raise ValueError("output buffer must match the query")
    if out is not None and any(ext.share_bytes(out, tensor) for tensor in (
            query, key_cache, value_cache, block_tables, context_lens, workspace) if tensor is not None):
        raise ValueError("output buffer must not overlap the inputs or the workspace")
    if validate:
        for length, table in zip(context_lens.tolist(), block_tables.tolist()):
            if not 0 < length <= width * block_size:
                raise ValueError("invalid context length")
            if any(page < 0 or page >= num_blocks for page in table[:-(-length // block_size)]):
                raise ValueError("physical block id out of range")
    _need_hip(query)
    query = _dense(query)
    if out is None:
        out = torch.empty_like(query)
    lib = ext.load_hip_extension()
    need = lib.fp4_workspace_size(batch, q_heads, kv_heads, head_dim, block_size, width, partition_tokens)
    ws_ptr, ws_bytes, workspace = _workspace(workspace, need, query.device)
    with torch.cuda.device(query.device):
        lib.call("mvme_fp4_paged_attention", out.data_ptr(), query.data_ptr(), key_cache.data_ptr(),
                 value_cache.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), batch, q_heads, kv_heads,
                 head_dim, num_blocks, block_size, width, partition_tokens, ext.dtype_code(query.dtype), ws_ptr,
                 ws_bytes, ext.current_stream(query.device))
    return out


def _dense(query):
    """The query with dense 16-byte aligned rows."""
    query = query.contiguous()
    return query.clone() if query.data_ptr() % 16 else query


def _workspace(workspace, need, device):
    """(address, bytes, owner) of the caller's workspace, or of a new one."""
    if workspace is None:
        if not need:
            return None, 0, None
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif workspace.device != device or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous tensor on the query's device")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace


def fp4_prefill_workspace_bytes(num_seqs, total_tokens, q_heads, kv_heads, head_dim, block_size, table_width,
                                chunk_tokens=0):
    """Bytes of the key-chunk workspace paged_prefill_attention_fp4 needs for these shapes (0: none)."""
    return ext.load_hip_extension().fp4_prefill_workspace_size(num_seqs, total_tokens, q_heads, kv_heads, head_dim,
                                                               block_size, table_width, chunk_tokens)


def paged_prefill_attention_fp4(q, key_cache, value_cache, cu_seqlens_q, query_starts, block_tables, context_lens,
                                block_size, *, backend="hip", validate=True, chunk_tokens=0, workspace=None):
    """Packed causal queries over a packed KV cache: ``paged_prefill_attention`` on 4-bit pages.

    q [total_queries, Hq, D] fp16/bf16; sequence s owns rows
    ``[cu_seqlens_q[s], cu_seqlens_q[s + 1])``, row i of it sits at position
    ``query_starts[s] + i`` and sees the keys up to it; the chunk's own keys
    are read from the cache, so they are written first.  Rows that see no key
    and rows behind the last sequence are zeros.  A NaN block, of a value too,
    makes the rows that see its key NaN in all dims (decode keeps a value's to
    its 32).  ``validate=False`` reads no metadata on the host.
    ``chunk_tokens`` (0 = library plan) splits keys over work-groups;
    ``workspace`` may supply the buffer for it.  The plan goes by the width of
    ``block_tables``: pass them as wide as the longest context needs, and few
    rows behind the last sequence (clearing them is slow).
    """
    _backend(backend, "prefill")
    if not validate and workspace is None:
        result = ext.native.fp4_prefill(q, key_cache, value_cache, cu_seqlens_q, query_starts, block_tables,
                                        context_lens, block_size, chunk_tokens)
        if result is not None:
            return result
    if q.dtype not in _HALF:
        raise ValueError("HIP paged prefill requires HIP FP16/BF16")
    if q.ndim != 3 or q.shape[1] <= 0:
        raise ValueError("paged prefill Q must be [tokens, heads, head_dim] with divisible GQA heads")
    tokens, q_heads, head_dim = q.shape
    if head_dim not in HEAD_DIMS:
        raise ValueError("packed attention supports head_dim 32,64,96,128,192,256")
    _check_caches(key_cache, value_cache, block_size, head_dim)
    num_blocks, kv_heads, _ = key_cache.shape
    if q_heads % kv_heads:
        raise ValueError("paged prefill Q must be [tokens, heads, head_dim] with divisible GQA heads")
    metadata = (cu_seqlens_q, query_starts, block_tables, context_lens)
    if (cu_seqlens_q.ndim != 1 or query_starts.ndim != 1 or context_lens.ndim != 1 or block_tables.ndim != 2
            or block_tables.shape[0] <= 0 or block_tables.shape[1] <= 0
            or query_starts.numel() != block_tables.shape[0] or context_lens.numel() != block_tables.shape[0]
            or cu_seqlens_q.numel() != block_tables.shape[0] + 1):
        raise ValueError("paged prefill metadata shapes do not match request count")
    if any(t.dtype != torch.int64 or not t.is_contiguous() for t in metadata):
        raise ValueError("paged prefill metadata must be contiguous int64 tensors")
    width = block_tables.shape[1]
    if width * block_size > MAX_TABLE_CAPACITY:
        raise ValueError("maximum table capacity is 1M tokens")
    if type(chunk_tokens) is not int or chunk_tokens < 0:
        raise ValueError("chunk_tokens must be a nonnegative integer")
    _check_devices(q, (key_cache, value_cache, *metadata))
    if validate:
        offsets, starts, tables, lengths = (t.tolist() for t in metadata)
        if offsets[0] != 0 or offsets[-1] != tokens or any(b < a for a, b in zip(offsets, offsets[1:])):
            raise ValueError("query offsets must be monotone and cover all packed queries")
        for index, (start, length, table) in enumerate(zip(starts, lengths, tables)):
            count = offsets[index + 1] - offsets[index]
            if start < 0 or length != start + count or length > len(table) * block_size:
                raise ValueError("query start/context length exceeds block table capacity or query range")
            if any(page < 0 or page >= num_blocks for page in table[:-(-length // block_size)]):
                raise ValueError("active block table contains an invalid physical page")
    _need_hip(q)
    q = _dense(q)
    output = torch.empty_like(q)
    if tokens == 0:
        return output
    lib = ext.load_hip_extension()
    num_seqs = query_starts.numel()
    need = lib.fp4_prefill_workspace_size(num_seqs, tokens, q_heads, kv_heads, head_dim, block_size, width,
                                          chunk_tokens)
    ws_ptr, ws_bytes, workspace = _workspace(workspace, need, q.device)
    with torch.cuda.device(q.device):
        lib.call("mvme_fp4_paged_prefill_attention", output.data_ptr(), q.data_ptr(), key_cache.data_ptr(),
                 value_cache.data_ptr(), cu_seqlens_q.data_ptr(), query_starts.data_ptr(), block_tables.data_ptr(),
                 context_lens.data_ptr(), num_seqs, tokens, q_heads, kv_heads, head_dim, num_blocks, block_size,
                 width, chunk_tokens, ext.dtype_code(q.dtype), ws_ptr, ws_bytes, ext.current_stream(q.device))
    return output
