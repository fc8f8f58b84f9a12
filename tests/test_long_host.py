"""The operators for long contexts on the CPU: refusals, page bookkeeping, the C ABI's argument checks."""

from pathlib import Path
import re

import pytest
import torch

import long_cases as lc
from mini_engine_hip.cache import KVCachePool, PagePool
from mini_engine_hip.kernels import hip_extension as ext
from mini_engine_hip.kernels.evict import evict_kv_cache
from mini_engine_hip.kernels.shared import _check_groups, paged_attention_shared_prefix
from mini_engine_hip.kernels.weights import check_weights, paged_attention_weights, prefill_attention_weights

HEADER = Path(__file__).resolve().parents[1] / "include" / "mvme_long.h"


@pytest.fixture(scope="module")
def lib():
    return ext.load_hip_extension()


def test_library_exports_every_declared_symbol(lib):
    names = re.findall(r"^(?:size_t|int) (mvme_\w+)\(", HEADER.read_text(), re.M)
    assert sorted(names) == sorted(ext.LONG_SIGNATURES)
    for name in names:
        assert hasattr(lib._lib, name)


# ---------------------------------------------------------------------------
# Pages.
# ---------------------------------------------------------------------------
def test_truncate_gives_back_pages_behind_the_tokens():
    pool = PagePool(10, 16)
    table = pool.allocate("a", 100)  # seven pages
    assert pool.truncate("a", 33) == table[:3] and pool.free_blocks == 7
    assert pool.truncate("a", 33) == table[:3]
    assert pool.extend("a", 64) == table[:4]  # the page given back last comes out first
    assert pool.truncate("a", 0) == [] and pool.free_blocks == 10
    with pytest.raises(ValueError):
        pool.truncate("a", 1)
    with pytest.raises(ValueError):
        pool.truncate("a", -1)


def test_truncate_keeps_pages_that_others_hold():
    pool = PagePool(10, 16)
    prefix = pool.allocate("system", 48)
    pool.allocate_with_prefix("a", 80, prefix)
    pool.truncate("a", 16)
    assert pool.table("a") == prefix[:1] and pool.refcount(prefix[1]) == 1 and pool.free_blocks == 7
    pool.free("system")
    assert pool.free_blocks == 9 and pool.refcount(prefix[0]) == 1


# ---------------------------------------------------------------------------
# Shared prefixes.
# ---------------------------------------------------------------------------
def test_groups_are_checked():
    tables = torch.tensor([[1, 2, 3], [1, 2, 4], [1, 5, 6], [-1, -1, -1]])
    lens = torch.tensor([40, 48, 20, 0])

    def check(offsets, prefixes):
        _check_groups(tables, lens, torch.tensor(offsets), torch.tensor(prefixes), 16)

    check([0, 2], [32])
    check([0, 2, 4], [32, 0])
    check([0, 4], [32])          # the third and fourth are too short to share
    check([3, 4], [32])          # nobody has the prefix
    for offsets, prefixes, word in (([0, 3], [17], "same pages"), ([0, 2], [33], "same pages"), ([0, 5], [16], "rise"),
                                    ([2, 1], [16], "rise"), ([-1, 2], [16], "rise"), ([0, 2], [49], "capacity"),
                                    ([0, 2], [-1], "capacity")):
        with pytest.raises(RuntimeError, match=word):
            check(offsets, prefixes)


def test_shared_prefix_refusals():
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    cache = torch.zeros(3, 16, 2, 64, dtype=torch.float16)
    tables, lens = torch.zeros(2, 2, dtype=torch.int64), torch.ones(2, dtype=torch.int64)
    offsets, prefixes = torch.tensor([0, 2]), torch.tensor([16])

    def call(**kw):
        named = {"query": q, "offsets": offsets, "prefixes": prefixes, "backend": "hip", **kw}
        paged_attention_shared_prefix(named["query"], cache, cache, tables, lens, 16, named["offsets"], named["prefixes"],
                                      backend=named["backend"], validate=False)

    for kw, error in (({"backend": "torch"}, ValueError), ({"query": q.float()}, ValueError),
                      ({"offsets": torch.tensor([0])}, ValueError), ({"offsets": torch.tensor([0, 1, 2])}, ValueError),
                      ({"prefixes": torch.tensor([16], dtype=torch.int32)}, ValueError),
                      ({"offsets": torch.tensor([0, 1, 2, 2]), "prefixes": torch.tensor([1, 1, 1])}, ValueError),
                      ({}, RuntimeError)):  # CPU tensors
        with pytest.raises(error):
            call(**kw)


# ---------------------------------------------------------------------------
# Weights.
# ---------------------------------------------------------------------------
def test_weights_are_checked():
    good = torch.zeros(2, 3, 40)
    check_weights(good, (2, 3), 40, good.device)
    check_weights(good, (2, 3), 33, good.device)
    for bad, lines, capacity in ((good, (2, 3), 41), (good, (2, 4), 40), (good[0], (2, 3), 40), (good.half(), (2, 3), 40),
                                 (good.double(), (2, 3), 40), (good[..., :38], (2, 3), 30), (good, (2,), 40)):
        with pytest.raises(ValueError):
            check_weights(bad, lines, capacity, good.device)


def test_weights_entry_points_refuse():
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    cache = torch.zeros(3, 16, 2, 64, dtype=torch.float16)
    tables, lens = torch.zeros(2, 2, dtype=torch.int64), torch.ones(2, dtype=torch.int64)
    weights = torch.zeros(2, 2, 32)
    with pytest.raises(ValueError, match="backend"):
        paged_attention_weights(q, cache, cache, tables, lens, 16, weights, backend="torch")
    with pytest.raises(ValueError, match="FP16/BF16"):
        paged_attention_weights(q.float(), cache, cache, tables, lens, 16, weights)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_attention_weights(q, cache, cache, tables, lens, 16, weights)
    cu = torch.tensor([0, 1, 2])
    good = {"q": q, "key_cache": cache, "cu_seqlens_q": cu, "query_starts": lens - 1, "block_tables": tables,
            "context_lens": lens, "block_size": 16, "weights": weights}
    for change, word in (({"backend": "torch"}, "backend"), ({"q": q.float()}, "FP16/BF16"), ({"q": q[0]}, "tokens"),
                         ({"key_cache": cache.bfloat16()}, "type"), ({"block_size": 8}, "block size"),
                         ({"q": q[:, :3].contiguous()}, "GQA"), ({"q": q[..., :48].contiguous()}, "head"),
                         ({"cu_seqlens_q": cu[:2]}, "request count"), ({"query_starts": lens.int()}, "int64"),
                         ({"weights": weights[..., :31].contiguous()}, "capacity"), ({"weights": weights.half()}, "FP32"),
                         ({"cu_seqlens_q": torch.tensor([0, 2, 1])}, "monotone"),
                         ({"query_starts": lens}, "query range"), ({"block_tables": tables - 1}, "physical page"),
                         ({}, "HIP device")):
        with pytest.raises(ValueError, match=word):
            prefill_attention_weights(**{**good, **change})


# ---------------------------------------------------------------------------
# Eviction.
# ---------------------------------------------------------------------------
def evict_args(**kw):
    cache = torch.zeros(8, 16, 2, 64, dtype=torch.float16)
    args = {"key_cache": cache, "value_cache": cache.clone(), "weights": torch.zeros(2, 2, 48),
            "block_tables": torch.tensor([[0, 1, 2], [3, 4, 5]]), "context_lens": torch.tensor([40, 48]), "block_size": 16,
            "keep": 20}
    return {**args, **kw}


def test_eviction_refusals():
    cache = evict_args()["key_cache"]
    tables = evict_args()["block_tables"]
    for change, word in (({"backend": "torch"}, "backend"), ({"key_cache": cache[0]}, "contiguous"),
                         ({"value_cache": cache.bfloat16()}, "FP16/BF16"), ({"block_size": 8}, "block size"),
                         ({"key_cache": cache[..., :60].contiguous(), "value_cache": cache[..., :60].contiguous()}, "multiple of 8"),
                         ({"block_tables": tables[:1]}, "batch"), ({"context_lens": torch.tensor([40, 48], dtype=torch.int32)}, "int64"),
                         ({"first": torch.tensor([1])}, "first"), ({"keep": 0}, "keep"), ({"keep": 2.0}, "keep"), ({"keep": True}, "keep"),
                         ({"recent": -1}, "recent"), ({"weights": torch.zeros(2, 2, 47)}, "capacity"),
                         ({"weights": torch.zeros(1, 2, 2, 48)}, "weights"), ({"weights": torch.zeros(2, 2, 48).half()}, "FP32"),
                         ({"value_cache": cache, "key_cache": cache}, "overlap"),
                         ({"context_lens": torch.tensor([40, 49])}, "context length"), ({"context_lens": torch.tensor([0, 4])}, "context length"),
                         ({"block_tables": torch.tensor([[0, 1, 8], [3, 4, 5]])}, "physical"),
                         ({"first": torch.tensor([-1, 0])}, "first"),
                         ({"block_tables": torch.tensor([[0, 1, 2], [1, 4, 5]])}, "another sequence"),
                         ({"block_tables": torch.tensor([[0, 1, 2], [0, 4, 5]])}, "another sequence"),
                         ({"block_tables": torch.tensor([[0, 1, 0], [3, 4, 5]])}, "twice"), ({}, "HIP device")):
        with pytest.raises(ValueError, match=word):
            evict_kv_cache(**evict_args(**change))


def test_eviction_allows_protected_shared_pages():
    shared = torch.tensor([[0, 1, 2], [0, 4, 5]])
    with pytest.raises(ValueError, match="HIP device"):  # everything else was accepted
        evict_kv_cache(**evict_args(block_tables=shared, first=torch.tensor([16, 16])))
    with pytest.raises(ValueError, match="another sequence"):
        evict_kv_cache(**evict_args(block_tables=shared, first=torch.tensor([16, 15])))
    with pytest.raises(ValueError, match="HIP device"):  # behind the kept rows nothing is written
        evict_kv_cache(**evict_args(block_tables=torch.tensor([[0, 1, 2], [3, 4, 2]])))
    with pytest.raises(ValueError, match="HIP device"):  # nobody is over the bound
        evict_kv_cache(**evict_args(block_tables=shared, keep=48))


def test_pool_of_the_cpu_is_refused():
    with pytest.raises(ValueError):
        KVCachePool(1, 1, 16, 1, 64, device="cpu")


def test_reference_eviction():
    # The tests' own oracle, by hand: ties to the lowest position, NaN first, what is protected.
    w = torch.tensor([[[[5.0, 1.0, 1.0, float("nan"), -0.0, 0.0, 1.0, 9.0]]]])
    assert lc.evict(w, [8], 3)[0][0][0] == [0, 3, 7]
    assert lc.evict(w, [8], 5)[0][0][0] == [0, 1, 2, 3, 7]
    assert lc.evict(w, [8], 3, first=[2])[0][0][0] == [0, 1, 3]
    assert lc.evict(w, [7], 3, recent=2)[0][0][0] == [3, 5, 6]
    assert lc.evict(w, [6], 4, first=[3], recent=9)[0][0][0] == [0, 1, 2, 5]
    assert lc.evict(w, [4], 4)[0][0][0] == [0, 1, 2, 3]


# ---------------------------------------------------------------------------
# The C ABI.  (No launch: arguments are refused before.)
# ---------------------------------------------------------------------------
FAKE = 1 << 20  # an aligned address that nothing reads


def shared_call(lib, **kw):
    a = {"out": FAKE, "query": FAKE, "key": FAKE, "value": FAKE, "tables": FAKE, "lens": FAKE, "offsets": FAKE, "prefixes": FAKE,
         "batch": 64, "groups": 1, "q_heads": 16, "kv_heads": 8, "dim": 128, "blocks": 999, "block": 16, "width": 256, "always": 0,
         "dtype": 1, "ws": FAKE, "bytes": 1 << 40, "stream": None, **kw}
    return lib._lib.mvme_paged_attention_shared_prefix(*a.values())


@pytest.mark.parametrize("change,word", [
    ({"dtype": 2}, "FP16"), ({"batch": 0}, "empty"), ({"kv_heads": 3}, "GQA"), ({"dim": 100}, "head_dim"), ({"block": 0}, "table"),
    ({"width": 65537}, "1M"), ({"groups": -1}, "groups"), ({"groups": 65}, "groups"), ({"query": None}, "null"),
    ({"offsets": None}, "null"), ({"key": FAKE + 8}, "aligned"), ({"out": FAKE + 4}, "aligned"), ({"ws": None}, "workspace"),
    ({"bytes": 1000}, "workspace"), ({"ws": FAKE + 8}, "workspace"), ({"blocks": 1 << 31}, "too large"),
    ({"batch": 1 << 24, "q_heads": 8}, "too large"), ({"batch": 1 << 17, "width": 65536}, "too many")])
def test_shared_prefix_arguments(lib, change, word):
    assert shared_call(lib, **change) in (ext.EINVAL, ext.EWORKSPACE)
    assert word in lib.last_error()


def test_workspace_sizes(lib):
    # Few cached tokens: what paged attention needs.  Many: pieces of 16 and of 128 rows, D + 2 numbers each.
    assert lib.shared_prefix_workspace_size(4, 16, 8, 128, 1, 16, 35, 0) == lib.workspace_size(4, 16, 8, 128, 16, 35, 0)
    size = lib.shared_prefix_workspace_size(64, 16, 8, 128, 1, 16, 256, 0)
    assert size == ((8 * (1 + 1) + 512) * 128 + (8 * (2 + 64) + 512) * 16) * 130 * 4
    assert lib.shared_prefix_workspace_size(4, 16, 8, 128, 1, 16, 35, 1) > 0
    assert lib.shared_prefix_workspace_size(4, 16, 8, 100, 1, 16, 35, 0) == 0
    assert lib.shared_prefix_workspace_size(4, 16, 8, 128, 5, 16, 35, 0) == 0
    # Short or many sequences are whole; others keep 4 bytes per head and token.
    assert lib.weights_workspace_size(1, 16, 8, 128, 16, 32) == 0
    assert lib.weights_workspace_size(16, 16, 8, 128, 16, 256) == 0
    assert lib.weights_workspace_size(4, 16, 8, 128, 16, 256) > 4 * 16 * 4096 * 4
    assert lib.weights_workspace_size(1, 16, 8, 100, 16, 32) == 0
    assert lib.prefill_weights_workspace_size(1, 0, 16, 8, 128, 16, 32) == 0
    assert lib.prefill_weights_workspace_size(1, 32, 16, 8, 128, 16, 512) == 32 * 16 * 32 * 8
    assert lib.prefill_weights_workspace_size(1, 32, 16, 8, 100, 16, 512) == 0


@pytest.mark.parametrize("change,word", [
    ({"dtype": 3}, "FP16"), ({"layers": 0}, "empty"), ({"dim": 12}, "head_dim"), ({"dim": 1032}, "head_dim"), ({"width": 0}, "table"),
    ({"width": 65537}, "1M"), ({"row": 511}, "capacity"), ({"keep": 0}, "keep"), ({"recent": -1}, "recent"), ({"key": None}, "null"),
    ({"value": FAKE + 4}, "aligned"), ({"layers": 1 << 20, "batch": 1 << 10}, "too large"), ({"blocks": 1 << 40}, "too large")])
def test_eviction_arguments(lib, change, word):
    a = {"key": FAKE, "value": FAKE, "weights": FAKE, "new": FAKE, "row": 512, "kept": FAKE, "lens_out": FAKE, "tables": FAKE,
         "lens": FAKE, "first": None, "layers": 28, "batch": 64, "kv_heads": 8, "dim": 128, "blocks": 99, "block": 16, "width": 32,
         "keep": 100, "recent": 0, "dtype": 0, "stream": None, **change}
    assert lib._lib.mvme_evict_kv_cache(*a.values()) == ext.EINVAL
    assert word in lib.last_error()


@pytest.mark.parametrize("change,word", [({"row": 511}, "capacity"), ({"weights": None}, "null"), ({"width": 257, "row": 1 << 20, "ws": None}, "workspace"),
                                         ({"query": FAKE + 2}, "aligned"), ({"q_heads": 9}, "GQA")])
def test_weighted_step_arguments(lib, change, word):
    a = {"out": FAKE, "query": FAKE, "key": FAKE, "value": FAKE, "tables": FAKE, "lens": FAKE, "weights": FAKE, "row": 512, "batch": 1,
         "q_heads": 16, "kv_heads": 8, "dim": 128, "blocks": 99, "block": 16, "width": 32, "dtype": 0, "ws": FAKE, "bytes": 1 << 40,
         "stream": None, **change}
    assert lib._lib.mvme_paged_attention_weights(*a.values()) in (ext.EINVAL, ext.EWORKSPACE)
    assert word in lib.last_error()


@pytest.mark.parametrize("change,word", [({"row": 511}, "capacity"), ({"q": None}, "null"), ({"bytes": 8}, "workspace"), ({"dim": 48}, "head_dim"),
                                         ({"tokens": -1}, "empty"), ({"tokens": 1 << 31}, "too many"), ({"key": FAKE + 2}, "aligned")])
def test_prompt_arguments(lib, change, word):
    a = {"q": FAKE, "key": FAKE, "cu": FAKE, "starts": FAKE, "tables": FAKE, "lens": FAKE, "weights": FAKE, "row": 512, "seqs": 2,
         "tokens": 100, "q_heads": 16, "kv_heads": 8, "dim": 128, "blocks": 99, "block": 16, "width": 32, "dtype": 0, "ws": FAKE,
         "bytes": 1 << 40, "stream": None, **change}
    assert lib._lib.mvme_prefill_attention_weights(*a.values()) in (ext.EINVAL, ext.EWORKSPACE)
    assert word in lib.last_error()
