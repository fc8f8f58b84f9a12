"""Attention weights that cached tokens receive, ``backend="hip"``.

A request whose cache is bounded keeps an account of the attention that each
cached token received: fp32 ``[sequences, kv_heads, capacity]``, one number for
the query heads that share a kv head.  ``prefill_attention_weights`` adds what a
prompt's queries give (all of them, or the last ones), and
``paged_attention_weights`` is a decode step's attention that adds its own.
``kernels/evict.py`` drops the tokens that received least.
"""

from __future__ import annotations

import torch

from . import hip_extension as ext
from .paged import MAX_TABLE_CAPACITY, SUPPORTED_HEAD_DIMS, _check, _native_checks
from .shared import check_aligned, check_output, dense_rows, take_workspace


def check_weights(weights, lines, capacity, device):
    """fp32 ``[*lines, >= capacity]``, contiguous."""
    if (weights.ndim != len(lines) + 1 or tuple(weights.shape[:-1]) != tuple(lines) or weights.shape[-1] < capacity):
        raise ValueError("weights must be [sequences, kv_heads, at least the tables' capacity]")
    if weights.dtype != torch.float32 or not weights.is_contiguous():
        raise ValueError("weights must be a contiguous FP32 tensor")
    if weights.device != device:
        raise ValueError("weights must share the cache device")


def weights_workspace_bytes(batch, q_heads, kv_heads, head_dim, block_size, table_width):
    """Bytes of the workspace paged_attention_weights needs for these shapes."""
    return ext.load_hip_extension().weights_workspace_size(batch, q_heads, kv_heads, head_dim, block_size, table_width)


def paged_attention_weights(query, key_cache, value_cache, block_tables, context_lens, block_size, weights, *,
                            backend="hip", validate=True, out=None, workspace=None):
    """``paged_attention``, adding to ``weights`` the probability that each cached token receives.

    The first six arguments, the checks and the result are those of
    ``paged_attention``.  ``weights`` (fp32 ``[batch, kv_heads, S]``, S at least
    the tables' capacity) is changed in place: entry ``[b, h, j]`` grows by the
    sum over the query heads of kv head h, for ``j < context_lens[b]``; the
    others stay.  Autograd does not see it.  ``out`` / ``workspace`` may supply
    the buffers (``weights_workspace_bytes``: four bytes per query head and
    token of the tables' capacity, so pass tables as wide as the longest
    context needs).
    """
    if backend != "hip":
        raise ValueError("decode backend must be hip")
    if not validate and out is None and workspace is None:
        result = ext.native.decode_weights(query, key_cache, value_cache, block_tables, context_lens, block_size,
                                           weights)
        if result is not None:
            return result
    if query.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("HIP paged attention supports FP16/BF16")
    _native_checks(query, key_cache, value_cache, block_tables, context_lens, block_size, validate)
    check_aligned(key_cache, value_cache)
    batch, q_heads, head_dim = query.shape
    num_blocks, _, kv_heads, _ = key_cache.shape
    width = block_tables.shape[1]
    check_weights(weights, (batch, kv_heads), width * block_size, query.device)
    _check(not any(ext.share_bytes(weights, t) for t in (query, key_cache, value_cache, block_tables, context_lens,
                                                         workspace) if t is not None),
           "weights must not overlap the inputs or the workspace")
    if out is None:
        out = torch.empty_like(query)
    else:
        check_output(out, query, (query, key_cache, value_cache, block_tables, context_lens, weights, workspace))
    query = dense_rows(query)
    lib = ext.load_hip_extension()
    need = lib.weights_workspace_size(batch, q_heads, kv_heads, head_dim, block_size, width)
    with torch.cuda.device(query.device):
        ws_ptr, ws_bytes, workspace = take_workspace(workspace, need, query.device)
        lib.call("mvme_paged_attention_weights", out.data_ptr(), query.data_ptr(), key_cache.data_ptr(),
                 value_cache.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), weights.data_ptr(),
                 weights.shape[-1], batch, q_heads, kv_heads, head_dim, num_blocks, block_size, width,
                 ext.dtype_code(query.dtype), ws_ptr, ws_bytes, ext.current_stream(query.device))
    return out


def prefill_weights_workspace_bytes(num_seqs, total_tokens, q_heads, kv_heads, head_dim, block_size, table_width):
    """Bytes of the workspace prefill_attention_weights needs for these shapes."""
    return ext.load_hip_extension().prefill_weights_workspace_size(num_seqs, total_tokens, q_heads, kv_heads, head_dim,
                                                                   block_size, table_width)


def prefill_attention_weights(q, key_cache, cu_seqlens_q, query_starts, block_tables, context_lens, block_size, weights,
                              *, backend="hip", validate=True, workspace=None):
    """Add to ``weights`` the probability that a prompt's queries give each cached token.

    q [total_queries, Hq, D] and the metadata are those of
    ``paged_prefill_attention``: row i of sequence s sits at position
    ``query_starts[s] + i`` and sees the keys up to it, which are read from the
    cache.  They may be all rows of a prompt or its last ones.  ``weights``
    (fp32 ``[sequences, kv_heads, S]``, S at least the tables' capacity) is
    changed in place; autograd does not see it.  Nothing is returned.
    ``validate=False`` reads no metadata on the host: rows that no sequence
    owns, and sequences whose start or length cannot be, add nothing.
    """
    if backend != "hip":
        raise ValueError("paged prefill backend must be hip")
    if not validate and workspace is None:
        if ext.native.prefill_weights(q, key_cache, cu_seqlens_q, query_starts, block_tables, context_lens, block_size,
                                      weights):
            return
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("HIP paged prefill requires HIP FP16/BF16")
    if q.ndim != 3 or key_cache.ndim != 4 or q.shape[1] <= 0 or any(size <= 0 for size in key_cache.shape):
        raise ValueError("paged prefill Q must be [tokens, heads, head_dim] and the cache [pages, block, kv_heads, head_dim]")
    tokens, q_heads, head_dim = q.shape
    num_blocks, _, kv_heads, _ = key_cache.shape
    if key_cache.dtype != q.dtype or not key_cache.is_contiguous():
        raise ValueError("paged prefill K cache must be contiguous in the query's type")
    if key_cache.shape[1] != block_size or block_size <= 0:
        raise ValueError("block size mismatch")
    if head_dim not in SUPPORTED_HEAD_DIMS or key_cache.shape[3] != head_dim or q_heads % kv_heads:
        raise ValueError("head dimension or GQA mismatch (supported head_dim: 16,32,64,80,96,128,192,256)")
    metadata = (cu_seqlens_q, query_starts, block_tables, context_lens)
    if (cu_seqlens_q.ndim != 1 or query_starts.ndim != 1 or context_lens.ndim != 1 or block_tables.ndim != 2
            or block_tables.shape[0] <= 0 or block_tables.shape[1] <= 0
            or query_starts.numel() != block_tables.shape[0] or context_lens.numel() != block_tables.shape[0]
            or cu_seqlens_q.numel() != block_tables.shape[0] + 1):
        raise ValueError("paged prefill metadata shapes do not match request count")
    if any(t.dtype != torch.int64 or not t.is_contiguous() for t in metadata):
        raise ValueError("paged prefill metadata must be contiguous int64 tensors")
    width, num_seqs = block_tables.shape[1], block_tables.shape[0]
    if width * block_size > MAX_TABLE_CAPACITY:
        raise ValueError("maximum table capacity is 1M tokens")
    if any(t.device != q.device for t in (key_cache, *metadata)):
        raise ValueError("paged prefill tensors must share a device")
    check_weights(weights, (num_seqs, kv_heads), width * block_size, q.device)
    if any(ext.share_bytes(weights, t) for t in (q, key_cache, *metadata, workspace) if t is not None):
        raise ValueError("weights must not overlap the inputs or the workspace")
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
    if q.device.type != "cuda":
        raise ValueError("HIP paged prefill requires a HIP device")
    check_aligned(key_cache)
    if tokens == 0:
        return
    q = dense_rows(q.contiguous())
    lib = ext.load_hip_extension()
    need = lib.prefill_weights_workspace_size(num_seqs, tokens, q_heads, kv_heads, head_dim, block_size, width)
    with torch.cuda.device(q.device):
        ws_ptr, ws_bytes, workspace = take_workspace(workspace, need, q.device)
        lib.call("mvme_prefill_attention_weights", q.data_ptr(), key_cache.data_ptr(), cu_seqlens_q.data_ptr(),
                 query_starts.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), weights.data_ptr(),
                 weights.shape[-1], num_seqs, tokens, q_heads, kv_heads, head_dim, num_blocks, block_size, width,
                 ext.dtype_code(q.dtype), ws_ptr, ws_bytes, ext.current_stream(q.device))
