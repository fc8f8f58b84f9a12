"""Decode attention over shared prefixes, ``backend="hip"``.

Sequences that begin with the same pages (a cached system prompt attached to
several requests, the children of a fork) are attended together: each group's
prefix is read once for all its query heads, and what a sequence has of its own
once for its own.  Arguments, validation and errors follow ``paged_attention``.
"""

from __future__ import annotations

import torch

from . import hip_extension as ext
from .paged import _check, _native_checks


def check_aligned(*tensors):
    _check(all(t.data_ptr() % 16 == 0 for t in tensors), "KV caches must be 16-byte aligned")


def dense_rows(query):
    """The query at a 16-byte boundary (a slice of a larger tensor may begin between two)."""
    return query.clone() if query.data_ptr() % 16 else query


def take_workspace(workspace, need, device):
    """(address, bytes, owner) of the caller's workspace, or of a new one."""
    if workspace is None and not need:
        return None, 0, None
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    else:
        _check(workspace.device == device and workspace.is_contiguous(),
               "workspace must be a contiguous tensor on the query's device")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace


def check_output(out, query, others):
    _check(out.shape == query.shape and out.dtype == query.dtype and out.is_contiguous()
           and out.device == query.device, "output buffer must match the query")
    _check(not any(ext.share_bytes(out, t) for t in others if t is not None),
           "output buffer must not overlap the inputs or the workspace")
    _check(out.data_ptr() % 8 == 0, "output buffer must be 8-byte aligned")


def shared_prefix_workspace_bytes(batch, q_heads, kv_heads, head_dim, groups, block_size, table_width,
                                  always_share=False):
    """Bytes of the workspace paged_attention_shared_prefix needs for these shapes (0: none)."""
    return ext.load_hip_extension().shared_prefix_workspace_size(batch, q_heads, kv_heads, head_dim, groups, block_size,
                                                                 table_width, int(always_share))


def _check_groups(tables, lengths, offsets, prefixes, block_size):
    """Host-synchronising checks of the groups."""
    rows, spans, lens = offsets.tolist(), prefixes.tolist(), lengths.tolist()
    _check(rows[0] >= 0 and rows[-1] <= len(lens) and all(a <= b for a, b in zip(rows, rows[1:])),
           "group offsets must rise within the batch")
    for first, last, prefix in zip(rows, rows[1:], spans):
        _check(0 <= prefix <= tables.shape[1] * block_size, "prefix length exceeds block table capacity")
        if first == last or prefix == 0:
            continue
        pages = -(-prefix // block_size)
        whole = [b for b in range(first, last) if lens[b] >= prefix]
        _check(not whole or bool((tables[whole, :pages] == tables[whole[0], :pages]).all()),
               "sequences of a group must have the prefix in the same pages")


def paged_attention_shared_prefix(query, key_cache, value_cache, block_tables, context_lens, block_size, group_offsets,
                                  prefix_lens, *, backend="hip", validate=True, always_share=False, out=None,
                                  workspace=None):
    """``paged_attention`` for a batch in which sequences share prefixes.

    The first six arguments are those of ``paged_attention`` (full block tables
    and lengths), and so are the results, to rounding.  Sequences
    ``group_offsets[g] .. group_offsets[g + 1] - 1`` (int64 [groups + 1], rising;
    what is in no group shares nothing) hold their first ``prefix_lens[g]``
    tokens (int64 [groups]; any number, whether or not a page ends there) in the
    same pages.  A sequence shorter than its group's prefix (an empty one of a
    padded batch) is attended on its own.
    Calls of few cached tokens run ``paged_attention``'s kernels, which are
    ahead there, unless ``always_share``; a large batch most of which shares
    nothing is about as fast with ``paged_attention`` itself.  Groups of more
    than 32 query rows per kv head round the probabilities to the inputs' type
    before they meet the values.  ``validate=True`` reads the metadata
    on the host, and refuses groups whose pages differ; with ``validate=False``
    (graph capture) the caller answers for that, lengths and pages that cannot
    be are absent, and offsets that cannot be leave every sequence on its own.
    ``out`` / ``workspace`` may supply the buffers
    (``shared_prefix_workspace_bytes``).
    """
    if backend != "hip":
        raise ValueError("decode backend must be hip")
    if not validate and not always_share and out is None and workspace is None:
        result = ext.native.shared_prefix(query, key_cache, value_cache, block_tables, context_lens, block_size,
                                          group_offsets, prefix_lens)
        if result is not None:
            return result
    if query.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("HIP paged attention supports FP16/BF16")
    if (group_offsets.ndim != 1 or prefix_lens.ndim != 1 or group_offsets.numel() != prefix_lens.numel() + 1
            or prefix_lens.numel() > query.shape[0]):
        raise ValueError("group offsets must be [groups + 1] and prefix lengths [groups], at most one per sequence")
    if any(t.dtype != torch.int64 or not t.is_contiguous() for t in (group_offsets, prefix_lens)):
        raise ValueError("group offsets and prefix lengths must be contiguous int64 tensors")
    _native_checks(query, key_cache, value_cache, block_tables, context_lens, block_size, validate)
    _check(group_offsets.device == query.device and prefix_lens.device == query.device,
           "all inputs must be on the same CUDA device")
    check_aligned(key_cache, value_cache)
    if validate:
        _check_groups(block_tables, context_lens, group_offsets, prefix_lens, block_size)
    batch, q_heads, head_dim = query.shape
    num_blocks, _, kv_heads, _ = key_cache.shape
    groups = prefix_lens.numel()
    if out is None:
        out = torch.empty_like(query)
    else:
        check_output(out, query, (query, key_cache, value_cache, block_tables, context_lens, group_offsets, prefix_lens,
                                  workspace))
    query = dense_rows(query)
    lib = ext.load_hip_extension()
    need = lib.shared_prefix_workspace_size(batch, q_heads, kv_heads, head_dim, groups, block_size,
                                            block_tables.shape[1], int(bool(always_share)))
    with torch.cuda.device(query.device):
        ws_ptr, ws_bytes, workspace = take_workspace(workspace, need, query.device)
        lib.call("mvme_paged_attention_shared_prefix", out.data_ptr(), query.data_ptr(), key_cache.data_ptr(),
                 value_cache.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), group_offsets.data_ptr(),
                 prefix_lens.data_ptr(), batch, groups, q_heads, kv_heads, head_dim, num_blocks, block_size,
                 block_tables.shape[1], int(bool(always_share)), ext.dtype_code(query.dtype), ws_ptr, ws_bytes,
                 ext.current_stream(query.device))
    return out
