"""Attention weights on the GPU against float64: decode steps and prompts."""

import pytest
import torch

import long_cases as lc
from mini_engine_hip.kernels.paged import paged_attention
from mini_engine_hip.kernels.weights import (paged_attention_weights, prefill_attention_weights,
                                             prefill_weights_workspace_bytes, weights_workspace_bytes)

pytestmark = pytest.mark.gpu
DEV = "cuda"
# A probability as the sum of two numbers of the type: the upper bits leave a step (2^-10, 2^-7), of which the second
# loses half a step of its own.
SPLIT = {torch.float16: 2.0 ** -21, torch.bfloat16: 2.0 ** -15}


def step_case(seed, lens, *, heads=16, kv=8, dim=128, block=16, dtype=torch.bfloat16, pad=0, more=0):
    gen = torch.Generator().manual_seed(seed)
    tables, pages = lc.shared_tables(gen, lens, block, pad=pad)
    key, value = lc.caches(gen, pages, block, kv, dim, dtype, tables, lens)
    query = torch.randn(len(lens), heads, dim, generator=gen).to(dtype)
    weights = torch.rand(len(lens), kv, tables.shape[1] * block + more, generator=gen)
    return (*(t.to(DEV) for t in (query, key, value, tables)), torch.tensor(lens, device=DEV), block, weights.to(DEV))


def check_step(args, **kw):
    query, key, value, tables, lens, block, weights = args
    before = weights.clone()
    out = paged_attention_weights(*args, **kw)
    want, bound, received, slack = lc.decode(query, key, value, tables, lens.tolist(), block, SPLIT[query.dtype])
    lc.assert_within(out, want, bound)
    lc.assert_weights(weights, before, received, slack)
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [16, 32, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("block", [16, 7])
def test_step_head_dims(dtype, dim, block):
    check_step(step_case(dim, [1, 31, 32, 33, 129, 700], heads=6, kv=2, dim=dim, block=block, dtype=dtype, more=5))


@pytest.mark.parametrize("heads,kv", [(8, 8), (16, 8), (7, 1), (32, 4), (34, 2), (64, 1)])
@pytest.mark.parametrize("lens", [[128], [1, 2, 3], [5000, 17], [300] * 70])
def test_step_head_groups_and_lengths(heads, kv, lens):
    check_step(step_case(heads, lens, heads=heads, kv=kv, dim=64, block=32))


@pytest.mark.parametrize("lens,block", [([30000], 256), ([4096] * 8, 16), ([1500 * i + 1 for i in range(9)], 24)])
def test_step_long(lens, block):
    check_step(step_case(len(lens), lens, block=block))


@pytest.mark.parametrize("lens,pad", [([40, 3000], 4000), ([1, 17], 65530), ([700] * 20, 300)])
def test_step_wide_tables(lens, pad):
    check_step(step_case(len(lens), lens, heads=8, kv=4, dim=64, pad=pad), validate=False)


def test_step_is_paged_attention():
    args = step_case(1, [500, 64, 1])
    out = check_step(args)
    assert (out.float() - paged_attention(*args[:6]).float()).abs().max() < 1.6e-2


def test_step_empty_sequences_and_absent_pages():
    args = list(step_case(2, [200, 100, 300, 40], pad=1))
    args[4] = torch.tensor([200, 0, 10 ** 7, -3], device=DEV)
    out = check_step(args, validate=False)
    assert not out[1:].any()
    args[3][0, 4], args[3][0, 12] = -1, 10 ** 12
    check_step(args, validate=False)
    args[3][0] = -1
    before = args[6].clone()
    assert not paged_attention_weights(*args, validate=False).any() and torch.equal(args[6], before)


@pytest.mark.parametrize("n", [200, 3000])
def test_step_nan_does_not_reach_absent_tokens(n):
    args = list(step_case(9, [n, 40]))
    args[0][0, 3] = float("nan")  # a head of kv head 1
    args[3][0, 5] = -1
    before = args[6].clone()
    paged_attention_weights(*args, validate=False)
    w, there = args[6][0, 1], torch.arange(args[6].shape[2], device=DEV)
    there = (there < n) & (there // 16 != 5)
    assert torch.isnan(w[there]).all() and torch.equal(w[~there], before[0, 1][~there])
    assert torch.isfinite(args[6][0, 0]).all() and torch.isfinite(args[6][1]).all()


def test_step_probabilities_add_up_over_steps():
    args = step_case(3, [257, 1000], heads=8, kv=2, dim=64)
    before = args[6].clone()
    for _ in range(10):
        paged_attention_weights(*args, validate=False)
    gained = (args[6] - before).double().sum(-1)
    # Ten steps of four heads: 40, to 10 additions of fp32 per token to numbers below 2.
    assert (gained - 40).abs().max() < 1000 * 10 * 2.0 ** -23


def test_step_repeats_bit_for_bit_in_graphs_that_share_a_workspace():
    a, b = step_case(4, [900, 30, 2500]), step_case(5, [1000] * 9, heads=8, kv=8)
    need = max(weights_workspace_bytes(3, 16, 8, 128, 16, a[3].shape[1]), weights_workspace_bytes(9, 8, 8, 128, 16, 63))
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    start = [x[6].clone() for x in (a, b)]
    want = []
    for x, w in zip((a, b), start):
        outs = paged_attention_weights(*x, validate=False)
        want.append((outs, x[6].clone()))
    graphs, outs = [], []
    for x in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention_weights(*x, validate=False, workspace=ws))
        graphs.append(graph)
    for _ in range(3):
        for x, w in zip((a, b), start):
            x[6].copy_(w)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for x, out, (o, w) in zip((a, b), outs, want):
            assert torch.equal(out, o) and torch.equal(x[6], w)
        x = step_case(6, [50])
        paged_attention_weights(*x)


def test_step_buffers_and_refusals():
    args = step_case(7, [100, 600])
    start = args[6].clone()
    want = paged_attention_weights(*args)
    after = args[6].clone()
    args[6].copy_(start)
    out = torch.empty_like(want)
    ws = torch.full((weights_workspace_bytes(2, 16, 8, 128, 16, 38),), 255, dtype=torch.uint8, device=DEV)
    assert paged_attention_weights(*args, out=out, workspace=ws) is out
    assert torch.equal(out, want) and torch.equal(args[6], after)
    with pytest.raises(RuntimeError, match="workspace too small"):
        paged_attention_weights(*args, workspace=ws[16:])
    with pytest.raises(ValueError, match="FP32"):
        paged_attention_weights(*args[:6], args[6].half(), validate=False)
    with pytest.raises(ValueError, match="capacity"):
        paged_attention_weights(*args[:6], args[6][..., :600].contiguous(), validate=False)
    with pytest.raises(RuntimeError, match="overlap"):
        paged_attention_weights(*args, out=args[0], validate=False)
    assert torch.equal(args[6], after)


# ---------------------------------------------------------------------------
# Prompts.
# ---------------------------------------------------------------------------
def prompt_case(seed, new, prior, *, heads=16, kv=8, dim=128, block=16, dtype=torch.bfloat16, pad=0, more=0, tail=0):
    lens = [n + p for n, p in zip(new, prior)]
    gen = torch.Generator().manual_seed(seed)
    tables, pages = lc.shared_tables(gen, lens, block, pad=pad)
    key, _ = lc.caches(gen, pages, block, kv, dim, dtype, tables, lens)
    q = torch.randn(sum(new) + tail, heads, dim, generator=gen).to(dtype)
    cu = torch.tensor([0] + new).cumsum(0)
    weights = torch.rand(len(lens), kv, tables.shape[1] * block + more, generator=gen)
    return (q.to(DEV), key.to(DEV), cu.to(DEV), torch.tensor(prior, device=DEV), tables.to(DEV),
            torch.tensor(lens, device=DEV), block, weights.to(DEV))


def check_prompt(args, **kw):
    q, key, cu, starts, tables, lens, block, weights = args
    before = weights.clone()
    assert prefill_attention_weights(*args, **kw) is None
    received, slack = lc.prompt(q, key, cu.tolist(), starts.tolist(), tables, lens.tolist(), block)
    lc.assert_weights(weights, before, received, slack)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [16, 32, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("block", [16, 7])
def test_prompt_head_dims(dtype, dim, block):
    check_prompt(prompt_case(dim, [40, 1, 130], [0, 77, 300], heads=6, kv=2, dim=dim, block=block, dtype=dtype, more=3))


@pytest.mark.parametrize("heads,kv", [(8, 8), (7, 1), (32, 4), (34, 2), (64, 1)])
@pytest.mark.parametrize("new,prior", [([1], [0]), ([1], [500]), ([64], [0]), ([65, 63], [63, 65]), ([200] * 5, [0] * 5)])
def test_prompt_shapes(heads, kv, new, prior):
    check_prompt(prompt_case(heads, new, prior, heads=heads, kv=kv, dim=64, block=32))


@pytest.mark.parametrize("new,prior,block", [([32], [8160], 16), ([2000], [0], 256), ([700, 5], [1000, 9000], 24),
                                             ([1], [30000], 256), ([20] * 70, [30 * i for i in range(70)], 16)])
def test_prompt_long(new, prior, block):
    check_prompt(prompt_case(len(new), new, prior, block=block))


@pytest.mark.parametrize("new,prior,pad", [([32], [500], 4000), ([3, 1000], [7, 0], 4000), ([1, 5], [0, 60], 65530),
                                           ([128] * 9, [50] * 9, 300)])
def test_prompt_wide_tables(new, prior, pad):
    check_prompt(prompt_case(len(new), new, prior, heads=8, kv=4, dim=64, pad=pad), validate=False)


def test_prompts_in_graphs_that_share_a_workspace():
    cases = [prompt_case(11, [100, 17], [400, 0]), prompt_case(12, [1500], [0], heads=8, kv=8)]
    need = [prefill_weights_workspace_bytes(x[3].numel(), x[0].shape[0], x[0].shape[1], x[1].shape[2], 128, 16, x[4].shape[1])
            for x in cases]
    ws = torch.empty(max(need), dtype=torch.uint8, device=DEV)
    start, want, graphs = [x[7].clone() for x in cases], [], []
    for x in cases:
        prefill_attention_weights(*x, validate=False)
        want.append(x[7].clone())
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            prefill_attention_weights(*x, validate=False, workspace=ws)
        graphs.append(graph)
    for _ in range(3):
        for x, w in zip(cases, start):
            x[7].copy_(w)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x[7], w) for x, w in zip(cases, want))
        ws.fill_(255)


def test_prompt_rows_that_no_sequence_owns_and_sequences_that_cannot_be():
    args = list(prompt_case(1, [30, 20, 10, 40], [100, 0, 50, 0], pad=1, tail=9))
    check_prompt(args, validate=False)
    args[3] = torch.tensor([100, -1, 60, 5], device=DEV)      # a negative start, one behind the context, rows past it
    check_prompt(args, validate=False)
    args[5] = torch.tensor([130, 0, 10 ** 9, 40], device=DEV)
    check_prompt(args, validate=False)


def test_prompt_absent_pages():
    args = list(prompt_case(2, [50, 50], [200, 0]))
    args[4][0, 2], args[4][0, 14], args[4][1, 0] = -1, 10 ** 10, -1
    check_prompt(args, validate=False)
    args[4][:] = -1
    before = args[7].clone()
    prefill_attention_weights(*args, validate=False)
    assert torch.equal(args[7], before)


def test_prompt_nan_reaches_what_its_row_sees():
    args = list(prompt_case(3, [100], [0], heads=2, kv=2, dim=64))
    args[0][40, 1] = float("nan")
    prefill_attention_weights(*args)
    w = args[7][0]
    assert torch.isfinite(w[0]).all() and torch.isnan(w[1, :41]).all() and torch.isfinite(w[1, 41:]).all()
    args = list(prompt_case(3, [100], [0], heads=2, kv=2, dim=64))
    args[0][40, 1] = float("nan")
    args[4][0, 1] = -1
    prefill_attention_weights(*args, validate=False)
    w = args[7][0, 1]
    assert torch.isnan(w[:16]).all() and torch.isfinite(w[16:32]).all() and torch.isnan(w[32:41]).all()


def test_prompt_large_scores():
    args = list(prompt_case(4, [300], [64], dtype=torch.float16))
    args[0] = args[0] * 30
    check_prompt(args)


def test_prompt_of_one_row_is_a_step():
    step = step_case(8, [700, 33])
    weights = step[6].clone()
    paged_attention_weights(*step)
    query, key, _, tables, lens, block, _ = step
    prefill_attention_weights(query, key, torch.arange(3, device=DEV), lens - 1, tables, lens, block, weights)
    # Both are fp32 sums of the same two probabilities.
    assert (weights - step[6]).abs().max() < 1e-5


def test_prompt_repeats_bit_for_bit_and_in_a_graph():
    args = prompt_case(5, [100, 17, 300], [400, 0, 0])
    start = args[7].clone()
    prefill_attention_weights(*args)
    want = args[7].clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        prefill_attention_weights(*args, validate=False)
    for _ in range(4):
        args[7].copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(args[7], want)
        other = prompt_case(6, [10], [10])
        prefill_attention_weights(*other)


def test_prompt_buffers_views_and_no_rows():
    args = list(prompt_case(7, [30, 20], [0, 70]))
    start = args[7].clone()
    prefill_attention_weights(*args)
    want = args[7].clone()
    ws = torch.full((prefill_weights_workspace_bytes(2, 50, 16, 8, 128, 16, args[4].shape[1]),), 255, dtype=torch.uint8,
                    device=DEV)
    args[7].copy_(start)
    prefill_attention_weights(*args, workspace=ws)
    assert torch.equal(args[7], want)
    wide = torch.zeros(50, 32, 128, dtype=args[0].dtype, device=DEV)
    wide[:, 5:21] = args[0]
    args[0] = wide[:, 5:21]
    args[7].copy_(start)
    prefill_attention_weights(*args, validate=False)
    assert torch.equal(args[7], want)
    with pytest.raises(RuntimeError, match="workspace too small"):
        prefill_attention_weights(*args, workspace=ws[16:])
    empty = prompt_case(8, [0, 0], [10, 20])
    before = empty[7].clone()
    prefill_attention_weights(*empty)
    assert torch.equal(empty[7], before)
