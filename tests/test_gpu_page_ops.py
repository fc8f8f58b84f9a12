"""Page copies and compaction on the GPU, bit for bit, and a packed cache's
whole life: write, fork, decode, compact, decode again."""

import pytest
import torch

import fp4_cases as f4
from mini_engine_hip.cache import KVCachePool, KVCachePoolFP4, PagePool
from mini_engine_hip.kernels.fp4 import (paged_attention_fp4, paged_prefill_attention_fp4, write_kv_cache_batch_fp4,
                                         write_kv_cache_slots_fp4)
from mini_engine_hip.kernels.pages import compact_kv_pages, copy_kv_pages
from mini_engine_hip.kernels.paged import paged_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


def noise(shape, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    size = torch.empty((), dtype=dtype).element_size()
    count = 1
    for n in shape:
        count *= n
    return torch.randint(0, 256, (count * size,), generator=gen, dtype=torch.uint8).view(dtype).view(shape).to(DEV)


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# Pages of 1, 2, 4, 12, 16 and more bytes, pieces that do not divide, one plane and many.
@pytest.mark.parametrize("shape,page_dim,dtype", [
    ((9, 1), 0, torch.uint8), ((9, 3), 0, torch.uint8), ((9, 3), 0, torch.float16), ((9, 3), 0, torch.int32),
    ((7, 2, 4, 8), 0, torch.bfloat16), ((2, 3, 9, 4, 2, 32), 2, torch.float16), ((2, 5, 8, 2, 1088), 2, torch.uint8),
    ((2, 9, 16, 8, 129), 1, torch.bfloat16), ((1, 2, 6, 256, 8, 128), 2, torch.bfloat16), ((6,), 0, torch.int64),
    ((3, 8, 100003), 1, torch.uint8),
])
def test_copies_are_bit_exact_and_touch_nothing_else(shape, page_dim, dtype):
    cache = noise(shape, dtype)
    pages = shape[page_dim]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1))
    for moves in (0, 1, pages // 2):
        src, dst = order[:moves], order[moves:2 * moves]
        want = cache.clone()
        index = (slice(None),) * page_dim
        want[(*index, dst.to(DEV))] = cache[(*index, src.to(DEV))]
        copy_kv_pages(cache, src.to(DEV), dst.to(DEV), page_dim=page_dim)
        assert same(cache, want)


def test_one_source_feeds_several_pages_and_absent_pages_are_skipped():
    cache = noise((2, 8, 4, 16), torch.bfloat16)
    want = cache.clone()
    want[:, 3] = want[:, 6] = cache[:, 1]
    copy_kv_pages(cache, torch.tensor([1, 1], device=DEV), torch.tensor([3, 6], device=DEV), page_dim=1)
    assert same(cache, want)
    src = torch.tensor([-1, 8, 2, 2, 1 << 40, 0], device=DEV)
    dst = torch.tensor([0, 1, -1, 9, 5, 7], device=DEV)
    want[:, 7] = cache[:, 0]
    copy_kv_pages(cache, src, dst, page_dim=1, validate=False)
    assert same(cache, want)


def test_cache_that_starts_off_alignment():
    for dtype, offset in ((torch.float16, 1), (torch.int32, 1), (torch.uint8, 5)):
        flat = noise((1 + 6 * 64 + 8,), dtype)
        before, cache = flat.clone(), flat[offset:offset + 6 * 64].view(6, 64)
        copy_kv_pages(cache, torch.tensor([5, 0], device=DEV), torch.tensor([2, 3], device=DEV))
        want = before.clone()
        page = want[offset:offset + 6 * 64].view(6, 64)
        page[2], page[3] = page[5].clone(), page[0].clone()
        assert same(flat, want)


@pytest.mark.parametrize("rows,width", [(1, 1), (3, 100), (64, 33)])
def test_compaction_renumbers_tables(rows, width):
    pages, moves = 50, 9
    cache = noise((2, pages, 64), torch.uint8)
    gen = torch.Generator().manual_seed(rows)
    src = torch.arange(pages - moves, pages)
    dst = torch.randperm(pages - moves, generator=gen)[:moves]
    tables = torch.randint(-1, pages, (rows, width), generator=gen)
    tables[0, 0] = pages + 5  # no page: stays
    want_cache, want_tables = cache.clone(), tables.clone()
    want_cache[:, dst.to(DEV)] = cache[:, src.to(DEV)]
    for s, d in zip(src.tolist(), dst.tolist()):
        want_tables[tables == s] = d
    dev = tables.to(DEV)
    compact_kv_pages(cache, src.to(DEV), dst.to(DEV), dev, page_dim=1)
    assert same(cache, want_cache) and torch.equal(dev.cpu(), want_tables)
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    compact_kv_pages(cache, none, none, dev, page_dim=1)
    compact_kv_pages(cache, src.to(DEV), dst.to(DEV), none, page_dim=1)  # no tables on the device
    assert same(cache, want_cache) and torch.equal(dev.cpu(), want_tables)


def test_pages_past_four_gigabytes():
    cache = torch.empty(2, 40000, 65536, dtype=torch.uint8, device=DEV)  # 5.2 GB in two planes
    ids = torch.tensor([39999, 0, 20000, 33333], device=DEV)
    cache[:, ids] = noise((2, 4, 65536), torch.uint8)
    want = cache[:, ids].clone()
    copy_kv_pages(cache, ids, ids - torch.tensor([1, -1, 1, 1], device=DEV), page_dim=1)
    assert same(cache[:, torch.tensor([39998, 1, 19999, 33332], device=DEV)], want) and same(cache[:, ids], want)


def test_copies_in_a_graph_follow_their_ids():
    cache = noise((3, 20, 4096), torch.uint8)
    tables = torch.arange(20, device=DEV)
    src, dst = torch.tensor([18, 19], device=DEV), torch.tensor([0, 1], device=DEV)
    compact_kv_pages(cache.clone(), src, dst, tables.clone(), page_dim=1, validate=False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        compact_kv_pages(cache, src, dst, tables, page_dim=1, validate=False)
    for s, d in (((3, 9), (4, 5)), ((10, 19), (2, 0)), ((7, 8), (6, 1))):
        src.copy_(torch.tensor(s))
        dst.copy_(torch.tensor(d))
        want, numbers = cache.clone(), tables.clone()
        compact_kv_pages(want, src, dst, numbers, page_dim=1, validate=False)
        graph.replay()
        torch.cuda.synchronize()
        assert same(cache, want) and torch.equal(tables, numbers)


def test_sixteen_bit_pool_forks_and_compacts():
    """A forked request decodes as its parent did; both do after a compaction."""
    gen = torch.Generator().manual_seed(2)
    pool, host = KVCachePool(2, 12, 16, 2, 64), PagePool(12, 16, order=[11, 3, 8, 0, 9, 1, 10, 2, 4, 5, 6, 7])
    pool.clear()
    table = host.allocate("a", 40)
    rows = [torch.randn(40, 2, 64, generator=gen).bfloat16().to(DEV) for _ in range(4)]
    for layer in range(2):
        pool.write_hip(layer, table, 0, rows[2 * layer], rows[2 * layer + 1])
    child, moves = host.fork("a", "b", 40)
    pool.copy_pages(moves)
    query = torch.randn(2, 4, 64, generator=gen).bfloat16().to(DEV)
    query[1] = query[0]
    tables = torch.tensor([table, child], device=DEV)
    lens = torch.tensor([40, 40], device=DEV)
    base = [paged_attention(query, *pool.layer(n), tables, lens, 16) for n in range(2)]
    assert all(torch.equal(out[0], out[1]) for out in base)
    moves = host.compact()
    assert moves
    pool.compact_pages(moves, tables)
    assert tables.tolist() == [host.table("a"), host.table("b")]
    again = [paged_attention(query, *pool.layer(n), tables, lens, 16) for n in range(2)]
    assert all(torch.equal(x, y) for x, y in zip(base, again))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_packed_pool_serves_forked_requests(dtype):
    """Prompt chunks, a fork, decode steps of both branches, a free, a compaction
    and more steps, with every attention against float64 on the rows written."""
    layers, block, kv, heads, dim, steps = 2, 16, 2, 4, 64, 20
    gen = torch.Generator().manual_seed(3)
    pool, host = KVCachePoolFP4(layers, 24, block, kv, dim), PagePool(24, block, order=list(range(23, -1, -1)))
    history = {}  # request -> per layer (keys, values) in float64

    def stored(rows):
        return f4.values(*f4.quantise(rows))

    def rows(count):
        return [[torch.randn(count, kv, dim, generator=gen).to(dtype) for _ in range(2)] for _ in range(layers)]

    def remember(request, new):
        old = history.get(request)
        history[request] = [[torch.cat((old[n][i], stored(new[n][i]))) if old else stored(new[n][i]) for i in range(2)]
                            for n in range(layers)]

    def check(outputs, layer, requests, query):
        for row, request in enumerate(requests):
            k, v = history[request][layer]
            for h in range(heads):
                want, bound = f4.attention(query[row, h].double(), k[:, h // 2], v[:, h // 2])
                f4.assert_within(outputs[row, h], want, bound)

    host.allocate("filler", 5 * block)
    host.allocate("a", 37 + 2 * steps)
    at = 0
    for count in (30, 7):  # the prompt in two chunks
        new = rows(count)
        table = torch.tensor(host.table("a"))
        slots = torch.arange(at, at + count)
        slots = table[slots // block] * block + slots % block
        remember("a", new)
        for n in range(layers):
            write_kv_cache_slots_fp4(*pool.layer(n), slots.to(DEV), new[n][0].to(DEV), new[n][1].to(DEV), block)
            query = torch.randn(count, heads, dim, generator=gen).to(dtype)
            out = paged_prefill_attention_fp4(query.to(DEV), *pool.layer(n), torch.tensor([0, count], device=DEV),
                                              torch.tensor([at], device=DEV), table[None].to(DEV),
                                              torch.tensor([at + count], device=DEV), block)
            for t in (0, count - 1):
                k, v = (x[:at + t + 1] for x in history["a"][n])
                for h in range(heads):
                    f4.assert_within(out[t, h], *f4.attention(query[t, h].double(), k[:, h // 2], v[:, h // 2]))
        at += count
    child, moves = host.fork("a", "b", at)
    assert moves
    pool.copy_pages(moves)
    history["b"] = [list(pair) for pair in history["a"]]
    tables = None
    requests = ["a", "b"]
    for step in range(steps):
        if step == 8:  # the filler ends: its pages are holes now
            host.free("filler")
            moves = host.compact()
            assert moves
            pool.compact_pages(moves, tables)
            assert [row[:len(host.table(r))] for row, r in zip(tables.tolist(), requests)] == [host.table(r) for r in requests]
        length = at + step + 1
        for request in requests:  # pages for the new token, private
            if length > len(host.table(request)) * block:
                break
            _, moves = host.make_writable(request, (length - 1) // block)
            pool.copy_pages(moves)
        else:
            width = max(len(host.table(r)) for r in requests)
            tables = torch.tensor([host.table(r) + [-1] * (width - len(host.table(r))) for r in requests], device=DEV)
            new = [rows(1) for _ in requests]
            lens = torch.tensor([length] * 2, device=DEV)
            query = torch.randn(2, heads, dim, generator=gen).to(dtype)
            for row, request in enumerate(requests):
                remember(request, new[row])
            for n in range(layers):
                key, value = (torch.cat([new[row][n][i] for row in range(2)]).to(DEV) for i in range(2))
                write_kv_cache_batch_fp4(*pool.layer(n), tables, lens - 1, key, value, block)
                check(paged_attention_fp4(query.to(DEV), *pool.layer(n), tables, lens, block), n, requests, query)
            continue
        break
    assert step > 8
    k, v = pool.gather(1, host.table("b"), at, dtype)
    assert torch.equal(k.cpu().double(), history["b"][1][0][:at]) and torch.equal(v.cpu().double(), history["b"][1][1][:at])


def test_more_pages_than_one_launch_has_work_groups():
    """A work-group a page and plane, 2^24 + 10 of them: a launch has at most 2^24 - 1 of 256 threads."""
    moves = (1 << 23) + 5
    cache = torch.randint(0, 256, (2, 2 * moves + 3, 16), dtype=torch.uint8, device=DEV)
    want = cache.clone()
    want[:, :moves] = cache[:, moves + 3:]
    dst = torch.arange(moves, device=DEV)
    tables = torch.tensor([[0, moves + 3, 2 * moves + 2, -1, moves + 1]], device=DEV)
    compact_kv_pages(cache, dst + moves + 3, dst, tables, page_dim=1, validate=False)
    assert torch.equal(cache, want) and tables.tolist() == [[0, 0, moves - 1, -1, moves + 1]]


@pytest.mark.parametrize("at", [32, 37])
def test_branches_of_a_fork_decode_pages_beyond_it(at):
    """A fork at a page boundary and behind one: both branches write 40 tokens, three new pages each, and every step
    is within the bounds of float64 on the rows written."""
    block, kv, heads, dim, steps, dtype = 16, 2, 4, 64, 40, torch.bfloat16
    gen = torch.Generator().manual_seed(at)
    pool, host = KVCachePoolFP4(1, 16, block, kv, dim), PagePool(16, block, order=list(range(15, -1, -1)))
    host.allocate("filler", 3 * block)
    table = host.allocate("a", at)
    prompt = [torch.randn(at, kv, dim, generator=gen).to(dtype) for _ in range(2)]
    pool.write_hip(0, table, 0, prompt[0].to(DEV), prompt[1].to(DEV))
    _, moves = host.fork("a", "b", at)
    assert len(moves) == (1 if at % block else 0)
    pool.copy_pages(moves)
    requests = ["a", "b"]
    history = {r: [f4.values(*f4.quantise(x)) for x in prompt] for r in requests}
    ran = 0
    for step in range(steps):
        length = at + step + 1
        for request in requests:
            host.extend(request, length)
            _, moves = host.make_writable(request, (length - 1) // block)
            assert not moves  # what a branch writes behind the fork is its own
        tables = torch.tensor([host.table(r) for r in requests], device=DEV)
        if step == 20:
            host.free("filler")
            moves = host.compact()
            assert moves
            pool.compact_pages(moves, tables)
            assert tables.tolist() == [host.table(r) for r in requests]
        new = [torch.randn(2, kv, dim, generator=gen).to(dtype) for _ in range(2)]
        lens = torch.tensor([length] * 2, device=DEV)
        write_kv_cache_batch_fp4(*pool.layer(0), tables, lens - 1, new[0].to(DEV), new[1].to(DEV), block)
        query = torch.randn(2, heads, dim, generator=gen).to(dtype)
        got = paged_attention_fp4(query.to(DEV), *pool.layer(0), tables, lens, block)
        for row, request in enumerate(requests):
            history[request] = [torch.cat((old, f4.values(*f4.quantise(x[row:row + 1]))))
                                for old, x in zip(history[request], new)]
            k, v = history[request]
            for h in range(heads):
                f4.assert_within(got[row, h], *f4.attention(query[row, h].double(), k[:, h // 2], v[:, h // 2]))
        ran += 1
    assert ran == steps and all(len(host.table(r)) == -(-(at + steps) // block) for r in requests)
    for request in requests:
        for rows, want in zip(pool.gather(0, host.table(request), at + steps, dtype), history[request]):
            assert torch.equal(rows.cpu().double(), want)
