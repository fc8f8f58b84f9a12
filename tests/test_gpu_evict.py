"""Eviction on the GPU against a sort, bit for bit, and a request's whole life:
prompt, account, eviction, shared-prefix decode, steps, eviction again."""

import pytest
import torch

import long_cases as lc
from mini_engine_hip.cache import KVCachePool, PagePool
from mini_engine_hip.kernels.evict import evict_kv_cache
from mini_engine_hip.kernels.shared import paged_attention_shared_prefix
from mini_engine_hip.kernels.weights import paged_attention_weights, prefill_attention_weights

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bits(t):
    return t.contiguous().view(torch.uint8)


def case(seed, lens, *, layers=2, kv=4, dim=64, block=16, dtype=torch.bfloat16, pad=0, more=0, levels=0):
    gen = torch.Generator().manual_seed(seed)
    tables, pages = lc.shared_tables(gen, lens, block, pad=pad)
    shape = (layers, pages, block, kv, dim)
    # Any bit pattern, NaN among them.
    key, value = (torch.randint(-32768, 32768, shape, generator=gen, dtype=torch.int16).view(dtype) for _ in range(2))
    row = (layers, len(lens), kv, tables.shape[1] * block + more)
    weights = torch.rand(row, generator=gen) if not levels else torch.randint(0, levels, row, generator=gen).float()
    return key.to(DEV), value.to(DEV), weights.to(DEV), tables.to(DEV), torch.tensor(lens, device=DEV), block


def check(args, keep, *, first=None, recent=0, **kw):
    key, value, weights, tables, lens, block = args
    before = [t.clone() for t in (key, value, weights)]
    first_dev = None if first is None else torch.tensor(first, device=DEV)
    kept, new_lens, new_weights = evict_kv_cache(*args, keep, first=first_dev, recent=recent, **kw)
    layers, batch, kv, row = weights.shape
    capacity = tables.shape[1] * block
    usable = [n if 0 < n <= capacity else 0 for n in lens.tolist()]
    chosen = lc.evict(before[2].cpu(), usable, keep, first, recent)
    want_kept = torch.full((layers, batch, kv, min(keep, row)), -1, dtype=torch.int64)
    want_weights = torch.zeros_like(before[2]).cpu()
    want_key, want_value = before[0].clone(), before[1].clone()
    w, pages = before[2].cpu(), tables.cpu()
    for l in range(layers):
        for b in range(batch):
            for h in range(kv):
                at = torch.tensor(chosen[l][b][h], dtype=torch.int64)
                want_kept[l, b, h, :len(at)] = at
                want_weights[l, b, h, :len(at)] = w[l, b, h, at]
                to = torch.arange(len(at))
                src, dst = pages[b, at // block], pages[b, to // block]
                there = (src >= 0) & (src < key.shape[1]) & (dst >= 0) & (dst < key.shape[1])
                at, to, src, dst = (t[there].to(DEV) for t in (at, to, src, dst))
                for old, new in ((before[0], want_key), (before[1], want_value)):
                    new[l, dst, to % block, h] = old[l, src, at % block, h]
    assert torch.equal(kept.cpu(), want_kept)
    assert torch.equal(bits(new_weights.cpu()), bits(want_weights))
    assert torch.equal(bits(key), bits(want_key)) and torch.equal(bits(value), bits(want_value))
    assert torch.equal(bits(weights), bits(before[2]))
    assert new_lens.tolist() == [min(n, keep) if u else n for n, u in zip(lens.tolist(), usable)]
    return kept, new_lens, new_weights


@pytest.mark.parametrize("dim", [8, 16, 24, 64, 80, 128, 192, 256, 1024])
@pytest.mark.parametrize("block", [16, 7])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_of_every_size(dim, block, dtype):
    check(case(dim, [100, 37, 60], kv=3, dim=dim, block=block, dtype=dtype, more=3), 50, first=[4, 0, 9], recent=11)


@pytest.mark.parametrize("keep", [1, 2, 63, 64, 65, 255, 256, 1000, 1299, 1300, 5000])
@pytest.mark.parametrize("levels", [0, 1, 3])
def test_bounds_and_ties(keep, levels):
    check(case(keep, [1300, 1, 700, 64], levels=levels), keep, first=[0, 3, 10, 64], recent=5)


@pytest.mark.parametrize("first,recent", [(0, 0), (0, 100), (100, 0), (60, 60), (99, 1), (1000, 1000), (0, 99), (1, 98)])
def test_what_is_protected(first, recent):
    check(case(first + recent, [400, 101, 100]), 100, first=[first] * 3, recent=recent)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 5000, 16384, 16385, 40000])
def test_long_sequences(n):
    check(case(n, [n], layers=1, kv=2, dim=32, block=32), n // 2 + 1, first=[3], recent=33)


@pytest.mark.parametrize("n", [513, 2048, 2049, 8192, 8193, 12000, 20000])
def test_long_rows_of_few_levels(n):
    check(case(n, [n, n - 1, n // 3], layers=1, kv=1, dim=8, block=1, levels=3), n // 2, first=[3, 0, 1], recent=7)
    check(case(n, [n, n - 1, n // 3], layers=1, kv=1, dim=8, block=1, levels=3), 10, first=[3, 10, 1], recent=9)


@pytest.mark.parametrize("pad", [200, 2000, 65000])
def test_wide_tables(pad):
    check(case(pad, [300, 50, 120], layers=1, kv=2, dim=16, pad=pad), 100, first=[0, 7, 30], recent=20)


def test_strange_weights():
    args = case(1, [300, 300, 300, 300], layers=1, kv=1, dim=8)
    w = args[2]
    w[0, 0, 0, ::3] = float("nan")
    w[0, 0, 0, 1::9] = float("-inf")
    w[0, 1, 0] = torch.where(torch.arange(w.shape[-1], device=DEV) % 2 == 0, -0.0, 0.0)
    w[0, 2, 0] = -w[0, 2, 0]
    w[0, 2, 0, 5::7] = float("inf")
    w[0, 3, 0] *= 1e-42  # subnormal
    for keep in (20, 120, 299):
        check([t.clone() if isinstance(t, torch.Tensor) else t for t in args], keep, recent=2)


def test_nothing_to_evict_and_lengths_that_cannot_be():
    args = list(case(2, [50, 60, 70, 80], pad=1))
    check(args, 100)
    check(args, 2 ** 70, recent=2 ** 70)
    check(args, 40, recent=2 ** 64 + 3)
    args = list(case(2, [50, 60, 70, 80], pad=1))
    args[4] = torch.tensor([0, -7, 10 ** 8, 80], device=DEV)
    check(args, 40, validate=False)


def test_rows_of_absent_pages_do_not_move():
    args = list(case(3, [200, 200]))
    args[3][0, 1], args[3][0, 9], args[3][1, 0] = -1, 10 ** 11, -1
    check(args, 90, recent=4, validate=False)


def test_one_layer_without_its_dimension():
    key, value, weights, tables, lens, block = case(4, [100, 40], layers=1)
    want = evict_kv_cache(key.clone(), value.clone(), weights, tables, lens, block, 30, recent=3)
    for validate in (True, False):
        k, v = key.clone()[0], value.clone()[0]
        got = evict_kv_cache(k, v, weights[0], tables, lens, block, 30, recent=3, validate=validate)
        assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2][0])


def test_pages_past_four_gigabytes():
    pages = 150000
    key, value = (torch.zeros(1, pages, 16, 8, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    tables = torch.tensor([[pages - 1, 5, pages - 70000, 140000, 9]], device=DEV)
    noise = torch.randn(2, 5, 16, 8, 128, device=DEV).bfloat16()
    key[0, tables[0]], value[0, tables[0]] = noise[0], noise[1]
    weights = torch.rand(1, 1, 8, 80, device=DEV)
    kept, lens, _ = evict_kv_cache(key, value, weights, tables, torch.tensor([75], device=DEV), 16, 40)
    for got, want in ((key[0, tables[0]], noise[0]), (value[0, tables[0]], noise[1])):
        rows, old = got.reshape(80, 8, 128), want.reshape(80, 8, 128)
        for h in range(8):
            assert torch.equal(rows[:40, h], old[kept[0, 0, h], h])
        assert torch.equal(rows[40:], old[40:])


def test_eviction_in_a_graph():
    args = case(5, [300, 150, 90])
    copies = [t.clone() for t in args[:3]]
    want = evict_kv_cache(copies[0].clone(), copies[1].clone(), *args[2:], 100, recent=7)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = evict_kv_cache(*args, 100, recent=7, validate=False)
    for _ in range(3):
        args[0].copy_(copies[0])
        args[1].copy_(copies[1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        evict_kv_cache(*case(6, [40]), 20)


def test_a_requests_whole_life():
    """Eight requests over one system prompt: their own prompts are weighed and trimmed, decoding goes on over the shared
    prefix, the steps add to the account, and the caches are trimmed again."""
    layers, heads, kv, dim, block, batch, prefix, keep = 2, 8, 4, 64, 16, 8, 64, 128
    dtype = torch.float16
    pages = PagePool(400, block, order=torch.randperm(400, generator=torch.Generator().manual_seed(1)).tolist())
    pool = KVCachePool(layers, 400, block, kv, dim, dtype=dtype)
    gen = torch.Generator(device=DEV).manual_seed(2)
    pool.key.normal_(generator=gen)
    pool.value.normal_(generator=gen)
    system = pages.allocate("system", prefix)
    lens = [prefix + 100 + 21 * b for b in range(batch)]
    width = -(-max(lens) // block) + 1
    for b, n in enumerate(lens):
        pages.allocate_with_prefix(f"r{b}", n, system)
    free = pages.free_blocks

    def tables():
        t = torch.full((batch, width), -1, dtype=torch.int64)
        for b in range(batch):
            own = pages.table(f"r{b}")
            t[b, :len(own)] = torch.tensor(own)
        return t.to(DEV)

    weights = torch.zeros(layers, batch, kv, width * block, device=DEV)
    window = 16
    starts = torch.tensor(lens, device=DEV) - window
    cu = torch.arange(batch + 1, device=DEV) * window
    now = torch.tensor(lens, device=DEV)
    for layer in range(layers):
        q = torch.randn(batch * window, heads, dim, generator=gen, device=DEV).to(dtype)
        prefill_attention_weights(q, pool.key[layer], cu, starts, tables(), now, block, weights[layer])
        received, slack = lc.prompt(q, pool.key[layer], cu.tolist(), starts.tolist(), tables(), lens, block)
        lc.assert_weights(weights[layer], torch.zeros_like(weights[layer]), received, slack)
    first = torch.full((batch,), prefix, device=DEV)
    for turn in range(2):
        args = (pool.key, pool.value, weights, tables(), now, block)
        kept, now, weights = check(args, keep, first=[prefix] * batch, recent=8)
        assert (kept[..., :prefix] == torch.arange(prefix, device=DEV)).all()
        for b, n in enumerate(now.tolist()):
            pages.truncate(f"r{b}", n)
        assert pages.free_blocks > free
        # One decode step over the shared prefix, and one more whose weights count.
        for layer in range(layers):
            query = torch.randn(batch, heads, dim, generator=gen, device=DEV).to(dtype)
            cache = pool.key[layer], pool.value[layer]
            out = paged_attention_shared_prefix(query, *cache, tables(), now, block, torch.tensor([0, batch], device=DEV),
                                                torch.tensor([prefix], device=DEV))
            want, bound, received, slack = lc.decode(query, *cache, tables(), now.tolist(), block, 2.0 ** -11)
            lc.assert_within(out, want, bound)
            before = weights[layer].clone()
            out = paged_attention_weights(query, *cache, tables(), now, block, weights[layer])
            lc.assert_within(out, want, bound)
            lc.assert_weights(weights[layer], before, received, slack)
        # The requests grow by twenty tokens, whose rows are what the pages hold.
        now = now + 20
        for b, n in enumerate(now.tolist()):
            pages.extend(f"r{b}", n)
    pages.free("system")
    for b in range(batch):
        pages.free(f"r{b}")
    assert pages.free_blocks == 400
