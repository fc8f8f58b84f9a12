"""Shared-prefix decode attention on the GPU against float64.

The calls are small, and so are made to share (``shared``); ``test_small_calls``
has the form that leaves it to the library.
"""

import functools

import pytest
import torch

import long_cases as lc
from mini_engine_hip.cache import PagePool
from mini_engine_hip.kernels.paged import paged_attention
from mini_engine_hip.kernels.shared import paged_attention_shared_prefix, shared_prefix_workspace_bytes

pytestmark = pytest.mark.gpu
DEV = "cuda"
shared = functools.partial(paged_attention_shared_prefix, always_share=True)


def case(seed, lens, groups, *, heads=16, kv=8, dim=128, block=16, dtype=torch.bfloat16, pad=0, poison=True):
    """groups: (first, last, prefix); what lies between them is in no group."""
    gen = torch.Generator().manual_seed(seed)
    tables, pages = lc.shared_tables(gen, lens, block, groups, pad=pad)
    key, value = lc.caches(gen, pages, block, kv, dim, dtype, tables, lens, poison)
    query = torch.randn(len(lens), heads, dim, generator=gen).to(dtype)
    offsets, prefixes = [0], []
    for first, last, prefix in groups:
        if first > offsets[-1]:  # a group that shares nothing fills the gap
            offsets.append(first)
            prefixes.append(0)
        offsets.append(last)
        prefixes.append(prefix)
    dev = [t.to(DEV) for t in (query, key, value, tables)]
    return (*dev, torch.tensor(lens, device=DEV), block, torch.tensor(offsets, device=DEV),
            torch.tensor(prefixes, dtype=torch.int64, device=DEV))


def check(args, **kw):
    out = shared(*args, **kw)
    query, key, value, tables, lens, block = args[:6]
    # (Where a prefix has more than 32 rows its probabilities are rounded once to the type.)
    want, bound, _, _ = lc.decode(query, key, value, tables, lens.tolist(), block, lc.HALF_STEP[query.dtype])
    lc.assert_within(out, want, bound)
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [16, 32, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("block", [16, 7])
def test_head_dims(dtype, dim, block):
    prefix = 100 // block * block
    # Narrow (5 sequences x 2 heads) and wide (20 x 2) groups, and two sequences alone.
    lens = [prefix + n for n in (0, 1, 40, 129, 3)] + [64] + [prefix + block + n for n in range(20)] + [1]
    check(case(dim, lens, [(0, 5, prefix), (6, 26, prefix + block)], heads=8, kv=4, dim=dim, block=block, dtype=dtype))


@pytest.mark.parametrize("heads,kv", [(8, 8), (16, 8), (14, 2), (7, 1), (32, 4), (34, 2), (40, 1)])
@pytest.mark.parametrize("batch", [2, 3, 17, 70])
def test_groups_of_heads(heads, kv, batch):
    lens = [256 + 37 * i % 300 for i in range(batch)]
    check(case(heads + batch, lens, [(0, batch, 256)], heads=heads, kv=kv, dim=64, block=32))


@pytest.mark.parametrize("prefix", [1, 15, 63, 64, 65, 127, 128, 129, 191, 640, 1000])
@pytest.mark.parametrize("batch", [4, 40])
def test_prefix_lengths(prefix, batch):
    # Pages of one token: the prefix may have any length.
    lens = [prefix + (i * 7) % 23 for i in range(batch)]
    check(case(prefix, lens, [(0, batch, prefix)], heads=4, kv=2, dim=64, block=1, dtype=torch.float16))


@pytest.mark.parametrize("block,prefix,batch", [(256, 2048, 12), (16, 6000, 6), (24, 4800, 33), (16, 20000, 3)])
def test_long_prefixes(block, prefix, batch):
    prefix = prefix // block * block
    lens = [prefix + 1 + 211 * i % 700 for i in range(batch)]
    check(case(batch, lens, [(0, batch, prefix)], block=block))


def test_several_groups_and_sequences_in_none():
    lens = [300 + i for i in range(10)] + [5, 900, 2000] + [1024 + 64 * i for i in range(30)] + [40] * 9
    check(case(3, lens, [(0, 10, 288), (13, 43, 1024), (44, 46, 32)]))


def test_many_groups_past_one_wave():
    lens = [32 + i % 50 for i in range(300)]
    groups = [(2 * i, 2 * i + 2, 32) for i in range(100)]
    check(case(4, lens, groups, heads=4, kv=2, dim=64))


def test_short_empty_and_single_members():
    # Shorter than the prefix, empty (a padded batch), alone in a group, longer than the table.
    lens = [200, 64, 63, 0, 128, 300, 1, 17, 0]
    args = list(case(5, lens, [(0, 6, 64), (6, 7, 0), (7, 8, 16)], pad=2))
    out = check(args, validate=False)
    assert not out[3].any() and not out[8].any()
    args[4] = args[4].clone()
    args[4][5], args[4][6] = 10 ** 6, -4
    out = check(args, validate=False)
    assert not out[5].any() and not out[6].any()


@pytest.mark.parametrize("batch", [6, 40, 100])
def test_first_members_of_a_group_may_be_padding(batch):
    # Empty rows with empty tables come first, and one too short.
    for empty in (1, 2, 70):
        if empty + 3 > batch:
            continue
        lens = [300 + i for i in range(batch)]
        args = list(case(20 + batch, lens, [(0, batch, 256)], heads=8, kv=4, dim=64))
        args[3], args[4] = args[3].clone(), args[4].clone()
        args[3][:empty], args[4][:empty] = -1, 0
        args[3][empty, 4:], args[4][empty] = -1, 60
        out = check(args, validate=False)
        assert not out[:empty].any() and out[empty:].any(-1).all()


def test_absent_pages_are_skipped():
    args = list(case(6, [500, 400, 333, 480], [(0, 4, 320)]))
    tables = args[3].clone()
    tables[:, 3], tables[:, 7] = -1, 10 ** 9   # in the prefix
    tables[2, 20] = -1                          # in a sequence's own part
    args[3] = tables
    check(args, validate=False)
    tables[:] = -1
    assert not shared(*args, validate=False).any()


def test_offsets_that_cannot_be_leave_sequences_on_their_own():
    args = list(case(7, [200] * 6, [(0, 6, 128)]))
    for offsets, prefixes in (([0, 9], [128]), ([4, 2], [128]), ([-1, 6], [128]), ([0, 6, 3, 6], [128, 128, 128]),
                              ([0, 6], [-5]), ([0, 6], [10 ** 9])):
        args[6] = torch.tensor(offsets, device=DEV)
        args[7] = torch.tensor(prefixes, device=DEV)
        check(args, validate=False)


@pytest.mark.parametrize("pad", [300, 4000, 65000])
def test_wide_tables(pad):
    check(case(30, [400, 333, 320, 500, 41], [(0, 4, 320)], heads=8, kv=4, dim=64, pad=pad))


def test_graphs_that_share_a_workspace():
    cases = [case(31, [900, 850, 1000], [(0, 3, 800)]), case(32, [300 + i for i in range(40)], [(0, 20, 256), (20, 40, 288)])]
    need = [shared_prefix_workspace_bytes(x[0].shape[0], 16, 8, 128, x[7].numel(), 16, x[3].shape[1], True) for x in cases]
    ws = torch.empty(max(need), dtype=torch.uint8, device=DEV)
    want, outs, graphs = [shared(*x) for x in cases], [], []
    for x in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(shared(*x, validate=False, workspace=ws))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        for out in outs:
            out.zero_()
        ws.fill_(255)


def test_no_groups_is_paged_attention():
    args = list(case(8, [1, 128, 129, 4000, 77], []))
    out = check(args)
    plain = paged_attention(*args[:6])
    assert (out.float() - plain.float()).abs().max() < 1.6e-2


def test_large_scores_and_infinite_values():
    args = list(case(9, [300] * 40, [(0, 40, 256)], dtype=torch.float16, poison=False))
    args[0] = args[0] * 40
    check(args)
    # A value that is infinite reaches all that see it, and no other sequence.  (As an infinity or as NaN: scores of this
    # size differ by more than 104, where exp() of the difference is 0 in fp32, and 0 times infinity is NaN.)
    page = int(args[3][7, 16])
    args[2][page, 3, 0, 5] = float("inf")
    out = shared(*args)
    assert not torch.isfinite(out[7, :2, 5]).any() and torch.isfinite(out[:7]).all() and torch.isfinite(out[8:]).all()


def test_nan_of_one_sequence_stays_there():
    args = list(case(10, [300] * 20 + [200] * 3, [(0, 20, 256)]))
    args[1][int(args[3][4, 16]), 2, 1] = float("nan")
    out = shared(*args)
    assert torch.isnan(out[4, 2:4]).all()
    out[4, 2:4] = 0
    assert torch.isfinite(out).all()


def test_results_do_not_change_from_call_to_call():
    args = case(11, [700 + 13 * i for i in range(50)], [(0, 50, 640)])
    first = shared(*args)
    for _ in range(5):
        assert torch.equal(shared(*args, validate=False), first)


def test_buffers_and_strange_alignment():
    args = list(case(12, [300] * 5, [(0, 5, 256)]))
    want = shared(*args)
    need = shared_prefix_workspace_bytes(5, 16, 8, 128, 1, 16, 19, True)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    out = torch.empty_like(want)
    assert shared(*args, out=out, workspace=ws) is out and torch.equal(out, want)
    flat = torch.empty(args[0].numel() + 1, dtype=args[0].dtype, device=DEV)
    flat[1:] = args[0].flatten()
    args[0] = flat[1:].view(args[0].shape)
    assert torch.equal(shared(*args), want)
    assert torch.equal(shared(*args, validate=False), want)
    with pytest.raises(RuntimeError, match="workspace too small"):
        shared(*args, workspace=ws[:need - 16])
    with pytest.raises(RuntimeError, match="overlap"):
        shared(*args, out=args[0])
    flat = torch.empty(args[1].numel() + 1, dtype=args[1].dtype, device=DEV)
    with pytest.raises(RuntimeError, match="aligned"):
        shared(args[0], flat[1:].view(args[1].shape), *args[2:], validate=False)


def test_pages_past_four_gigabytes():
    pages = 150000  # 4.9 GB of keys
    key, value = (torch.empty(pages, 16, 8, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    gen = torch.Generator().manual_seed(13)
    tables = torch.stack([torch.cat((torch.arange(4), torch.tensor([10 + b]))) for b in range(20)])
    tables = (pages - 1 - 7000 * tables).abs() % pages
    for b in range(20):
        for page in tables[b].tolist():
            key[page] = torch.randn(16, 8, 128, generator=gen).to(DEV)
            value[page] = torch.randn(16, 8, 128, generator=gen).to(DEV)
    query = torch.randn(20, 16, 128, generator=gen).to(torch.bfloat16).to(DEV)
    lens = torch.tensor([64 + 1 + b % 16 for b in range(20)], device=DEV)
    check((query, key, value, tables.to(DEV), lens, 16, torch.tensor([0, 20], device=DEV),
           torch.tensor([64], device=DEV)))


def test_graph_follows_its_metadata():
    batch = 24
    args = list(case(14, [600] * batch, [(0, batch, 512)], pad=3, poison=False))
    tables, lens, offsets, prefixes = args[3], args[4], args[6], args[7]
    shared(*args, validate=False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = shared(*args, validate=False)
    original = tables.clone()
    for n, last, prefix in ((600, 24, 512), (520, 24, 512), (601, 9, 256), (513, 0, 0), (600, 24, 64)):
        lens.fill_(n)
        lens[3] = 0
        offsets[1] = last
        prefixes.fill_(prefix)
        tables.copy_(original)
        graph.replay()
        torch.cuda.synchronize()
        want, bound, _, _ = lc.decode(*args[:4], lens.tolist(), args[5], 2.0 ** -8)
        lc.assert_within(out, want, bound)
        assert torch.equal(out, shared(*args, validate=False))


def test_two_streams_at_once():
    args = case(15, [900 + i for i in range(40)], [(0, 40, 896)])
    other = case(16, [300 + i for i in range(10)], [(0, 10, 256)], heads=8, kv=8, dim=64)
    want = [shared(*a) for a in (args, other)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(4):
        for a, stream in zip((args, other), streams):
            with torch.cuda.stream(stream):
                outs.append(shared(*a, validate=False))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, want[i % 2])


def test_small_calls():
    args = list(case(18, [300, 0, 290, 17], [(0, 3, 256)]))
    want, bound, _, _ = lc.decode(*args[:4], args[4].tolist(), 16, 2.0 ** -8)
    out = paged_attention_shared_prefix(*args, validate=False)
    lc.assert_within(out, want, bound)
    assert torch.equal(out, paged_attention(*args[:6], validate=False))
    assert torch.equal(out, paged_attention_shared_prefix(*args, validate=False, out=torch.empty_like(out)))


def test_large_calls_share_by_themselves():
    batch = 48
    args = case(19, [4096 + 30 + b for b in range(batch)], [(0, batch, 4096)])
    out = paged_attention_shared_prefix(*args, validate=False)
    assert torch.equal(out, shared(*args))
    check(args)


def test_forked_requests():
    pool = PagePool(64, 16)
    pool.allocate("parent", 200)
    for i in range(6):
        pool.fork("parent", f"child{i}", 192)
        pool.extend(f"child{i}", 192 + 5 * i + 1)
    lens = [200] + [193 + 5 * i for i in range(6)]
    names = ["parent"] + [f"child{i}" for i in range(6)]
    tables = torch.full((7, 14), -1, dtype=torch.int64)
    for b, name in enumerate(names):
        table = pool.table(name)
        tables[b, :len(table)] = torch.tensor(table)
    gen = torch.Generator().manual_seed(17)
    key, value = lc.caches(gen, 64, 16, 8, 128, torch.float16, tables, lens)
    query = torch.randn(7, 16, 128, generator=gen).half()
    check((*(t.to(DEV) for t in (query, key, value, tables)), torch.tensor(lens, device=DEV), 16,
           torch.tensor([0, 7], device=DEV), torch.tensor([192], device=DEV)))
