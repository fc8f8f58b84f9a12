"""What the packed cache's and the page operators' entry points refuse, in
Python and in the C ABI, before anything runs (CPU only)."""

import ctypes
from pathlib import Path
import re

import pytest
import torch

import fp4_cases as f4
from mini_engine_hip import build as hip_build
from mini_engine_hip.cache import KVCachePoolFP4
from mini_engine_hip.kernels import hip_extension as ext
from mini_engine_hip.kernels.fp4 import (fp4_record_bytes, gather_kv_cache_fp4, gather_kv_cache_slots_fp4,
                                         paged_attention_fp4, paged_prefill_attention_fp4, write_kv_cache_batch_fp4,
                                         write_kv_cache_slots_fp4)
from mini_engine_hip.kernels.pages import compact_kv_pages, copy_kv_pages

HEADER = Path(__file__).resolve().parents[1] / "include" / "mvme_fp4.h"


def ids(*values):
    return torch.tensor(values, dtype=torch.int64)


@pytest.fixture(scope="module")
def lib():
    return ext.load_hip_extension()


def test_library_exports_every_declared_symbol(lib):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    symbols = set(re.findall(r"\b(mvme_\w+)\s*\(", text))
    raw = ctypes.CDLL(str(hip_build.library_path()))
    assert all(hasattr(raw, name) for name in symbols)
    assert set(ext.PACKED_SIGNATURES) == symbols


def test_record_sizes_agree(lib):
    for block in (1, 7, 16, 256, 1000):
        for dim in range(32, 257, 32):
            size = f4.record_bytes(block, dim)
            assert fp4_record_bytes(block, dim) == size == lib._lib.mvme_fp4_record_bytes(block, dim)
    for block, dim in ((0, 64), (-1, 64), (16, 0), (16, 48), (16, 288), (1048577, 32), (16, 16), (16.0, 64)):
        with pytest.raises(ValueError):
            fp4_record_bytes(block, dim)
        assert type(block) is float or lib._lib.mvme_fp4_record_bytes(block, dim) == 0


def packed_inputs(dim=64, block=4, kv=2):
    cache = torch.zeros(6, kv, f4.record_bytes(block, dim), dtype=torch.uint8)
    rows = torch.randn(3, kv, dim).half()
    return cache, cache.clone(), rows, rows.clone(), block


def test_writes_refuse():
    kc, vc, key, value, block = packed_inputs()
    slots = ids(0, 9, 5)

    def refused(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            write_kv_cache_slots_fp4(*args, **kw)

    refused("backend", kc, vc, slots, key, value, block, backend="cuda")
    refused("block_size", kc, vc, slots, key, value, 0)
    refused("fp4_record_bytes", kc, vc, slots, key, value, 5)
    refused("fp4_record_bytes", kc, vc[:5], slots, key, value, block)
    refused("fp4_record_bytes", kc.int(), vc.int(), slots, key, value, block)
    refused("fp4_record_bytes", kc[::2], vc[::2], slots, key, value, block)
    refused("multiple of 32", kc, vc, slots, key[..., :48], value[..., :48], block)
    refused("matching the cache", kc, vc, slots, key[:, :1], value[:, :1], block)
    refused("matching the cache", kc, vc, slots, key, value[:2], block)
    refused("matching the cache", kc, vc, slots, key[0], value[0], block)
    refused("FP16/BF16", kc, vc, slots, key.float(), value.float(), block)
    refused("FP16/BF16", kc, vc, slots, key, value.bfloat16(), block)
    refused("int64", kc, vc, slots.int(), key, value, block)
    refused("int64", kc, vc, slots[:2], key, value, block)
    refused("capacity", kc, vc, ids(0, 24, 5), key, value, block)
    refused("capacity", kc, vc, ids(0, -1, 5), key, value, block)
    refused("duplicate", kc, vc, ids(0, 5, 5), key, value, block)
    refused("overlap", kc, kc, slots, key, value, block)
    alias = kc.view(-1)[:3 * 2 * 64 * 2].view(torch.float16).view(3, 2, 64)
    refused("overlap", kc, vc, slots, alias, value, block)
    refused("HIP device", kc, vc, slots, key, value, block)
    tables = ids(0, 1, 2, 3, 4, 5).view(3, 2)
    for match, args in (("shape mismatch", (kc, vc, tables[:2], slots, key, value, block)),
                        ("shape mismatch", (kc, vc, tables[:, :0], slots, key, value, block)),
                        ("shape mismatch", (kc, vc, tables, slots[:2], key, value, block)),
                        ("int64", (kc, vc, tables.int(), slots, key, value, block)),
                        ("int64", (kc, vc, tables.t().contiguous().t(), slots, key, value, block)),
                        ("offset out of range", (kc, vc, tables, ids(0, 8, 1), key, value, block)),
                        ("offset out of range", (kc, vc, tables, ids(0, -1, 1), key, value, block)),
                        ("physical block", (kc, vc, tables + 1, ids(0, 1, 7), key, value, block)),
                        ("duplicate", (kc, vc, tables * 0, ids(1, 1, 2), key, value, block)),
                        ("HIP device", (kc, vc, tables, ids(0, 7, 1), key, value, block))):
        with pytest.raises(ValueError, match=match):
            write_kv_cache_batch_fp4(*args)
    assert not kc.any() and not vc.any()


def test_reads_refuse():
    kc, vc, _, _, block = packed_inputs()
    for match, args in (("FP16/BF16", (kc, vc, ids(0), block, 64, torch.float32)),
                        ("int64", (kc, vc, ids(0).int(), block, 64, torch.float16)),
                        ("capacity", (kc, vc, ids(24), block, 64, torch.float16)),
                        ("fp4_record_bytes", (kc, vc, ids(0), block, 32, torch.float16)),
                        ("HIP device", (kc, vc, ids(0), block, 64, torch.float16))):
        with pytest.raises(ValueError, match=match):
            gather_kv_cache_slots_fp4(*args)
    for match, args in (("negative", (kc, vc, ids(0), -1, block, 64, torch.float16)),
                        ("exceeds", (kc, vc, ids(0), 5, block, 64, torch.float16)),
                        ("out of range", (kc, vc, ids(6), 4, block, 64, torch.float16)),
                        ("HIP device", (kc, vc, ids(0), 4, block, 64, torch.float16))):
        with pytest.raises(ValueError, match=match):
            gather_kv_cache_fp4(*args)


def test_attention_refuses():
    kc, vc, _, _, block = packed_inputs()
    query, tables, lens = torch.randn(2, 4, 64).half(), ids(0, 1, 2, 3).view(2, 2), ids(8, 3)

    def refused(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            paged_attention_fp4(*args, **kw)

    good = (query, kc, vc, tables, lens, block)
    refused("HIP device", *good)
    refused("backend", *good, backend="torch")
    refused("FP16/BF16", query.float(), *good[1:])
    refused("not empty", query[:0], kc, vc, tables[:0], lens[:0], block)
    refused("head_dim", query[..., :48], *good[1:])
    refused("head_dim", torch.randn(2, 4, 160).half(), *good[1:])
    refused("divisible", query[:, :3], *good[1:])
    refused("match the batch", query, kc, vc, tables[:1], lens, block)
    refused("match the batch", query, kc, vc, tables, lens[:1], block)
    refused("match the batch", query, kc, vc, tables[:, :0], lens, block)
    refused("int64", query, kc, vc, tables.int(), lens, block)
    refused("1M", query, kc, vc, torch.zeros(2, 262145, dtype=torch.int64), lens, block)
    refused("partition", *good, partition_tokens=-1)
    refused("partition", *good, partition_tokens=1.5)
    refused("output buffer", *good, out=torch.empty(2, 4, 32).half())
    refused("output buffer", *good, out=torch.empty(2, 4, 64).bfloat16())
    refused("context length", query, kc, vc, tables, ids(9, 3), block)
    refused("context length", query, kc, vc, tables, ids(0, 3), block)
    refused("physical block", query, kc, vc, ids(0, 6, 2, 3).view(2, 2), lens, block)
    refused("HIP device", query, kc, vc, ids(0, 1, 2, -1).view(2, 2), lens, block)  # padding behind the pages is fine

    q, cu, starts = torch.randn(5, 4, 64).half(), ids(0, 3, 5), ids(5, 1)
    good = (q, kc, vc, cu, starts, tables, lens, block)

    def prefill(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            paged_prefill_attention_fp4(*args, **kw)

    prefill("HIP device", *good)
    prefill("backend", *good, backend="cuda")
    prefill("FP16/BF16", q.float(), *good[1:])
    prefill("divisible", q[:, :3], *good[1:])
    prefill("divisible", q[0], *good[1:])
    prefill("head_dim", q[..., :16], *good[1:])
    prefill("request count", q, kc, vc, cu[:2], starts, tables, lens, block)
    prefill("request count", q, kc, vc, cu[:1], starts[:0], tables[:0], lens[:0], block)
    prefill("int64", q, kc, vc, cu, starts.int(), tables, lens, block)
    prefill("chunk_tokens", *good, chunk_tokens=-64)
    prefill("monotone", q, kc, vc, ids(0, 6, 5), starts, tables, lens, block)
    prefill("monotone", q, kc, vc, ids(0, 3, 4), starts, tables, lens, block)
    prefill("capacity or query range", q, kc, vc, cu, ids(4, 1), tables, lens, block)
    prefill("capacity or query range", q, kc, vc, cu, ids(-3, 1), tables, ids(0, 3), block)
    prefill("physical page", q, kc, vc, cu, starts, ids(0, -1, 2, 3).view(2, 2), lens, block)


def test_rounds_that_pass_32_bits(lib):
    """A million short sequences in tables of a million tokens: whole units by default, no partitions on request."""
    shape = (1 << 20, 8, 8, 128, 16, 65536)
    assert lib.fp4_workspace_size(*shape, 0) == 0
    with pytest.raises(RuntimeError, match="too many partitions"):
        lib.call("mvme_fp4_paged_attention", *[4096] * 6, *shape[:4], 64, *shape[4:], 1 << 19, 0, 4096, 1 << 40, None)
    assert lib.fp4_workspace_size(64, 8, 8, 128, 16, 65536, 0) > 0


def test_output_must_not_share_bytes_with_inputs():
    kc, vc, _, _, block = packed_inputs()
    query, tables, lens = torch.randn(2, 4, 64).half(), ids(0, 1, 2, 3).view(2, 2), ids(8, 3)
    size = 2 * 4 * 64
    for cache in (kc, vc):
        with pytest.raises(ValueError, match="overlap"):
            paged_attention_fp4(query, kc, vc, tables, lens, block,
                                out=cache.view(-1)[:2 * size].view(torch.float16).view(2, 4, 64))
    shared = torch.empty(4 * size, dtype=torch.uint8)
    with pytest.raises(ValueError, match="overlap"):
        paged_attention_fp4(query, kc, vc, tables, lens, block, workspace=shared,
                            out=shared[:2 * size].view(torch.float16).view(2, 4, 64))


def test_page_operators_refuse():
    cache = torch.zeros(2, 5, 4, 8)

    def refused(match, call, *args, **kw):
        with pytest.raises(ValueError, match=match):
            call(*args, **kw)

    for call, more in ((copy_kv_pages, ()), (compact_kv_pages, (ids(0, 4, -1),))):
        refused("backend", call, cache, ids(3), ids(0), *more, page_dim=1, backend="cuda")
        refused("page_dim", call, cache, ids(3), ids(0), *more, page_dim=4)
        refused("page_dim", call, cache, ids(3), ids(0), *more, page_dim=-1)
        refused("contiguous and not empty", call, cache.transpose(0, 1), ids(1), ids(0), *more)
        refused("contiguous and not empty", call, cache[:0], ids(1), ids(0), *more, page_dim=1)
        refused("int64", call, cache, ids(3).int(), ids(0), *more, page_dim=1)
        refused("pair up", call, cache, ids(3), ids(0, 1), *more, page_dim=1)
        refused("more moves", call, cache, ids(0, 0, 0), ids(1, 1, 1), *more, page_dim=0)
        refused("out of range", call, cache, ids(5), ids(0), *more, page_dim=1)
        refused("out of range", call, cache, ids(1), ids(-1), *more, page_dim=1)
        refused("two moves", call, cache, ids(3, 4), ids(0, 0), *more, page_dim=1)
        refused("both source", call, cache, ids(3, 4), ids(0, 3), *more, page_dim=1)
        refused("HIP device", call, cache, ids(3, 4), ids(1, 0), *more, page_dim=1)
    refused("rise", compact_kv_pages, cache, ids(4, 3), ids(0, 1), ids(4), page_dim=1)
    refused("int64", compact_kv_pages, cache, ids(3, 4), ids(0, 1), ids(4).int(), page_dim=1)
    src = ids(3, 4)
    refused("overlap", compact_kv_pages, cache, src, ids(0, 1), src, page_dim=1)
    refused("HIP device", copy_kv_pages, cache, ids(3, 3), ids(0, 1), page_dim=1)  # one source, two pages: fine


def test_packed_pool_refuses():
    with pytest.raises(ValueError, match="positive"):
        KVCachePoolFP4(1, 0, 16, 2, 64)
    with pytest.raises(ValueError, match="multiple of 32"):
        KVCachePoolFP4(1, 4, 16, 2, 80)
    with pytest.raises(ValueError, match="GPU"):
        KVCachePoolFP4(1, 4, 16, 2, 64, device="cpu")


def test_c_entry_points_refuse_before_launch(lib):
    def status(name, *args):
        return getattr(lib._lib, name)(*args)

    def write(kc=256, vc=256, pages=4, block=16, heads=8, dim=128, slots=8, key=16, value=16, tokens=4, ks=1024,
              vs=1024, dtype=1):
        return status("mvme_fp4_write_slots", kc, vc, pages, block, heads, dim, slots, key, value, tokens, ks, vs,
                      dtype, None)

    for args, message in (({"pages": 0}, "positive"), ({"heads": -1}, "positive"), ({"dim": 80}, "multiple of 32"),
                          ({"block": 0}, "multiple of 32"), ({"block": 1 << 21}, "multiple of 32"),
                          ({"dtype": 2}, "FP16/BF16"), ({"heads": 1 << 40}, "too large"), ({"pages": 1 << 60}, "too large"),
                          ({"tokens": -1}, "too many"), ({"tokens": 1 << 30}, "too many"), ({"kc": None}, "null"),
                          ({"slots": None}, "null"), ({"value": None}, "null"), ({"kc": 264}, "16-byte"),
                          ({"key": 17}, "2-byte"), ({"ks": 1000}, "stride")):
        assert write(**args) == ext.EINVAL and message in lib.last_error(), (args, lib.last_error())
    assert write(tokens=0, slots=None) == ext.OK
    assert status("mvme_fp4_write_batch", 256, 256, 4, 16, 8, 128, 8, 0, 8, 16, 16, 4, 1024, 1024, 1, None) == ext.EINVAL
    assert "table" in lib.last_error()
    assert status("mvme_fp4_write_batch", 256, 256, 4, 16, 8, 128, 8, 2, None, 16, 16, 4, 1024, 1024, 1, None) == ext.EINVAL
    assert status("mvme_fp4_gather_slots", 16, 16, 256, 256, 4, 16, 8, 100, 8, 4, 1, None) == ext.EINVAL
    assert status("mvme_fp4_gather", 16, 16, 256, 256, 4, 16, 8, 128, 8, 2, 33, 1, None) == ext.EINVAL
    assert "capacity" in lib.last_error()
    assert status("mvme_fp4_gather", 16, 16, 256, 256, 4, 16, 8, 128, 8, 2, 0, 1, None) == ext.OK

    def decode(out=16, query=16, kc=256, batch=2, heads=16, kv=8, dim=128, pages=4, block=16, width=2, part=0, dtype=1,
               ws=None, ws_bytes=0):
        return status("mvme_fp4_paged_attention", out, query, kc, 256, 8, 8, batch, heads, kv, dim, pages, block,
                      width, part, dtype, ws, ws_bytes, None)

    for args, message in (({"dtype": 7}, "FP16/BF16"), ({"batch": 0}, "empty"), ({"heads": 12}, "GQA"),
                          ({"dim": 160}, "head_dim"), ({"width": 0}, "block table"), ({"block": 0}, "block table"),
                          ({"width": 65537}, "1M"), ({"block": 1 << 40}, "1M"), ({"batch": 1 << 31}, "too large"),
                          ({"pages": 1 << 61}, "too large"), ({"out": None}, "null"), ({"query": 24}, "16-byte"),
                          ({"kc": 264}, "16-byte"), ({"part": -1}, "negative")):
        assert decode(**args) == ext.EINVAL and message in lib.last_error(), (args, lib.last_error())
    need = lib.fp4_workspace_size(2, 16, 8, 128, 16, 256, 64)
    assert need > 0
    assert decode(width=256, part=64, ws=256, ws_bytes=need - 1) == ext.EWORKSPACE and str(need) in lib.last_error()
    assert decode(width=256, part=64, ws=264, ws_bytes=need) == ext.EWORKSPACE
    assert lib.fp4_workspace_size(2, 16, 8, 160, 16, 256, 64) == 0
    assert lib.fp4_workspace_size(1 << 40, 1 << 40, 1, 128, 16, 256, 64) == 0
    assert lib.fp4_workspace_size(1, 16, 8, 128, 1 << 62, 4, 0) == 0

    def prefill(out=16, q=16, kc=256, seqs=2, total=40, heads=16, kv=8, dim=128, pages=4, block=16, width=2, chunk=0,
                dtype=1, ws=None, ws_bytes=0):
        return status("mvme_fp4_paged_prefill_attention", out, q, kc, 256, 8, 8, 8, 8, seqs, total, heads, kv, dim,
                      pages, block, width, chunk, dtype, ws, ws_bytes, None)

    for args, message in (({"dtype": 2}, "FP16/BF16"), ({"seqs": 0}, "empty"), ({"total": -1}, "empty"),
                          ({"kv": 3}, "GQA"), ({"dim": 16}, "head_dim"), ({"width": 65537}, "1M"),
                          ({"total": 1 << 40}, "too many"), ({"pages": 1 << 61}, "too large"), ({"chunk": -1}, "negative"),
                          ({"q": None}, "null"), ({"q": 8}, "16-byte"), ({"out": 4}, "8-byte")):
        assert prefill(**args) == ext.EINVAL and message in lib.last_error(), (args, lib.last_error())
    assert prefill(total=0) == ext.OK
    need = lib.fp4_prefill_workspace_size(2, 40, 16, 8, 128, 16, 256, 64)
    assert need > 0 and prefill(width=256, chunk=64, ws=256, ws_bytes=need - 1) == ext.EWORKSPACE

    def move(planes=16, count=2, pages=8, size=64, src=8, dst=8, moves=2, **kw):
        if kw:
            return status("mvme_compact_pages", planes, count, pages, size, src, dst, moves, kw["tables"], kw["entries"],
                          None)
        return status("mvme_copy_pages", planes, count, pages, size, src, dst, moves, None)

    for args, message in (({"count": 0}, "positive"), ({"pages": 0}, "positive"), ({"size": -1}, "positive"),
                          ({"size": 1 << 61}, "too large"), ({"moves": -1}, "more moves"), ({"moves": 9}, "more moves"),
                          ({"planes": None}, "null"), ({"src": None}, "null"), ({"dst": None}, "null"),
                          ({"tables": None, "entries": 4}, "null"), ({"tables": 8, "entries": -1}, "negative"),
                          ({"size": 1 << 40, "pages": 1 << 20, "moves": 1 << 20}, "too many")):
        assert move(**args) == ext.EINVAL and message in lib.last_error(), (args, lib.last_error())
    assert move(moves=0, src=None, dst=None) == ext.OK


def test_launches_that_do_not_fit_are_refused(lib):
    """A launch has at most 2^32 - 1 threads; what would need more, and so run short, is refused before it starts."""
    def decode(match, batch, heads, kv, dim, block, width, part):
        with pytest.raises(RuntimeError, match=match):
            lib.call("mvme_fp4_paged_attention", *[4096] * 6, batch, heads, kv, dim, 64, block, width, part, 0, 4096,
                     1 << 60, None)

    decode("head product too large", 1 << 24, 1, 1, 64, 16, 1, 0)       # a work-group of 256 threads per sequence
    decode("head product too large", 1 << 20, 256, 1, 64, 16, 1, 0)     # ... and 16 heads
    decode("too many partitions", 1 << 12, 1, 1, 64, 16, 1 << 16, 128)  # 2^25 rounds of 128 tokens
    decode("too many partitions", 1 << 21, 8, 1, 64, 16, 16, 128)       # the join has one per head

    def prefill(seqs, total, heads, kv, dim, width, chunk):
        with pytest.raises(RuntimeError, match="too many packed query rows"):
            lib.call("mvme_fp4_paged_prefill_attention", *[4096] * 8, seqs, total, heads, kv, dim, 64, 16, width, chunk,
                     0, 4096, 1 << 60, None)

    prefill(1 << 24, 1 << 24, 1, 1, 64, 1, 0)
    prefill(1, 1 << 20, 16, 1, 64, 1 << 16, 64)     # 2^17 row blocks, 2^14 chunks
    prefill(1, 1 << 20, 128, 1, 256, 8, 64)         # 2^25 joining work-groups of four rows


@pytest.mark.parametrize("tokens", [2 ** 63 - 1, 2 ** 63 - 127, 2 ** 63 - 128, 1024])
def test_partitions_and_chunks_of_any_size_leave_one(lib, tokens):
    """Sizes from the table's capacity on split nothing, up to the largest number that the calls take."""
    assert lib.fp4_workspace_size(2, 16, 8, 128, 16, 64, tokens) == 0
    assert lib.fp4_prefill_workspace_size(2, 40, 16, 8, 128, 16, 64, tokens) == 0
