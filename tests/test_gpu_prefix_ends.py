"""Shared-prefix attention on the GPU where the prefix ends inside a page or a
run of 16 tokens, against float64."""

import pytest
import torch

import long_cases as lc
from mini_engine_hip.cache import PagePool
from mini_engine_hip.kernels.shared import paged_attention_shared_prefix
from test_gpu_shared_prefix import check, shared

pytestmark = pytest.mark.gpu
DEV = "cuda"


def case(seed, lens, groups, *, heads=4, kv=2, dim=64, block=16, dtype=torch.bfloat16, pad=0):
    """groups: (first, last, prefix), one behind the other from sequence 0 on.  Members that have the whole prefix share
    all pages that it touches, its last one too; the others have pages of their own.  The page in which the first group's
    prefix ends is the cache's last, and all that no sequence holds is NaN."""
    gen = torch.Generator().manual_seed(seed)
    tables, pages = lc.shared_tables(gen, lens, block, extra=0, pad=pad)
    for first, last, prefix in groups:
        members = [b for b in range(first, last) if lens[b] >= prefix]
        for b in members:
            tables[b, :-(-prefix // block)] = tables[members[0], :-(-prefix // block)]
    first, last, prefix = groups[0]
    end = int(tables[next(b for b in range(first, last) if lens[b] >= prefix), (prefix - 1) // block])
    tables = torch.where(tables == end, pages - 1, torch.where(tables == pages - 1, end, tables))
    key, value = lc.caches(gen, pages, block, kv, dim, dtype, tables, lens)
    query = torch.randn(len(lens), heads, dim, generator=gen).to(dtype)
    dev = [t.to(DEV) for t in (query, key, value, tables)]
    return (*dev, torch.tensor(lens, device=DEV), block, torch.tensor([0] + [last for _, last, _ in groups], device=DEV),
            torch.tensor([prefix for _, _, prefix in groups], device=DEV))


@pytest.mark.parametrize("prefix", [1, 8, 15, 17, 24, 100, 1000, 1001, 1015])
@pytest.mark.parametrize("block", [16, 32, 48, 256])
@pytest.mark.parametrize("batch", [4, 40])
def test_prefixes_that_end_anywhere(prefix, block, batch):
    # Narrow (8 rows) and wide (80) groups; own parts of none, and over several page ends.
    lens = [prefix + (i * 37) % (3 * block + 50) for i in range(batch)]
    args = case(prefix + block, lens, [(0, batch, prefix)], block=block, dtype=torch.float16 if batch == 4 else torch.bfloat16)
    assert torch.equal(check(args), check(args, validate=False))


@pytest.mark.parametrize("dim", [16, 80, 128, 256])
@pytest.mark.parametrize("heads,kv", [(8, 8), (40, 1), (34, 2)])
def test_head_dims_and_groups(dim, heads, kv):
    lens = [100 + 29 * i for i in range(6)]
    check(case(dim + heads, lens, [(0, 6, 93)], heads=heads, kv=kv, dim=dim))


@pytest.mark.parametrize("batch", [5, 40])
def test_members_that_end_in_the_prefixs_last_run(batch):
    # 16 <= length < 24: shorter than the prefix, on pages of their own from the first token on.
    for short in (16, 17, 20, 23):
        lens = [short, 24, short, 60] + [24 + 7 * i % 90 for i in range(batch - 4)]
        args = case(short, lens, [(0, batch, 24)])
        assert args[3][0, 0] != args[3][1, 0]
        check(args)


def test_several_groups():
    lens = [40 + i % 50 for i in range(300)]
    check(case(3, lens, [(2 * i, 2 * i + 2, 17 + i % 24) for i in range(150)]))
    lens = [700 + i for i in range(90)]
    check(case(4, lens, [(0, 5, 333), (5, 45, 500), (45, 49, 15), (49, 90, 649)]))


def test_a_prefix_shorter_than_what_the_pages_share():
    pool = PagePool(64, 16)
    pool.allocate("parent", 200)
    names = ["parent"] + [f"child{i}" for i in range(6)]
    lens = [200] + [193 + 5 * i for i in range(6)]
    for name, n in zip(names[1:], lens[1:]):
        pool.fork("parent", name, 192)
        pool.extend(name, n)
    tables = torch.full((7, 14), -1, dtype=torch.int64)
    for b, name in enumerate(names):
        table = pool.table(name)
        tables[b, :len(table)] = torch.tensor(table)
    gen = torch.Generator().manual_seed(5)
    key, value = lc.caches(gen, 64, 16, 8, 128, torch.float16, tables, lens)
    query = torch.randn(7, 16, 128, generator=gen).half()
    for prefix in (192, 191, 177, 176, 175, 100, 16, 3):
        check((*(t.to(DEV) for t in (query, key, value, tables)), torch.tensor(lens, device=DEV), 16,
               torch.tensor([0, 7], device=DEV), torch.tensor([prefix], device=DEV)))


def test_large_calls_share_by_themselves():
    batch = 48
    args = case(6, [4001 + 3 * b for b in range(batch)], [(0, batch, 4001)], heads=16, kv=8, dim=128)
    out = paged_attention_shared_prefix(*args, validate=False)
    assert torch.equal(out, shared(*args))
    check(args)


def test_graph_follows_a_prefix_of_any_length():
    args = case(7, [600 + b for b in range(24)], [(0, 24, 512)], pad=3)
    lens, offsets, prefixes = args[4], args[6], args[7]
    shared(*args, validate=False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = shared(*args, validate=False)
    for prefix, last, n in ((512, 24, 600), (511, 24, 600), (300, 9, 600), (17, 24, 530), (500, 24, 505), (15, 24, 600), (512, 24, 590)):
        prefixes.fill_(prefix)
        offsets[1] = last
        lens.fill_(n)
        lens[3] = 0
        graph.replay()
        torch.cuda.synchronize()
        want, bound, _, _ = lc.decode(*args[:4], lens.tolist(), args[5], 2.0 ** -8)
        lc.assert_within(out, want, bound)
        assert torch.equal(out, shared(*args, validate=False))
