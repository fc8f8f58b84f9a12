"""The operators for long contexts in plain float64 torch: attention through
block tables, the weights that tokens receive, eviction; and the error bounds
that the kernels' tests use."""

from __future__ import annotations

import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rows_of(cache, table, n):
    """Rows of the tokens 0 .. n - 1 whose page exists, [tokens, kv_heads, dim] in float64, and their positions."""
    block, pages = cache.shape[1], cache.shape[0]
    pos = torch.arange(n, device=cache.device)
    page = table[pos // block]
    pos, page = pos[(page >= 0) & (page < pages)], page[(page >= 0) & (page < pages)]
    return cache[page, pos % block].double(), pos


def fp32_error(dim, size, n):
    """Relative error of a probability computed in fp32: a score is a sum of dim products no larger than `size` together,
    taken through one exponential; the divisor a sum over n keys in any order."""
    return 2.0 ** -23 * (2 * (dim + 8) * (size + 1) + n + 64)


def attention(query, key, value, weight_error):
    """Rows query [r, dim] over key / value [n, dim], float64 -> (outputs, bounds, probabilities, their bounds).

    A probability is off by `weight_error` of itself (its rounding for the
    value product) and what fp32 adds, and by 2^-32 of the largest at the
    smallest number of fp16 (2^-24, where the largest is 2^8 or more).
    """
    n, dim = key.shape
    if n == 0:
        zero = torch.zeros(query.shape[0], dim, dtype=torch.float64, device=query.device)
        return zero, zero, zero[:, :0], zero[:, :0]
    scores = query @ key.T / math.sqrt(dim)
    p = torch.softmax(scores, -1)
    size = (query.abs() @ key.abs().T / math.sqrt(dim)).amax(-1, keepdim=True)
    error = fp32_error(dim, size, n)
    lost = n * 2.0 ** -32 * value.abs().amax()
    return p @ value, (p @ value.abs()) * (weight_error + error) + lost, p, p * error


def decode(query, kc, vc, tables, lens, block, weight_error):
    """(outputs, bounds) [batch, heads, dim], (received, bounds) [batch, kv_heads, capacity]; float64, on kc's device."""
    batch, heads, dim = query.shape
    kv = kc.shape[2]
    group, capacity = heads // kv, tables.shape[1] * block
    outs, bounds = torch.zeros(2, batch, heads, dim, dtype=torch.float64, device=kc.device)
    received, slack = torch.zeros(2, batch, kv, capacity, dtype=torch.float64, device=kc.device)
    for b in range(batch):
        n = int(lens[b])
        if not 0 < n <= capacity:
            continue
        k, pos = rows_of(kc, tables[b], n)
        v, _ = rows_of(vc, tables[b], n)
        for h in range(kv):
            at = slice(h * group, (h + 1) * group)
            out, bound, p, off = attention(query[b, at].double(), k[:, h], v[:, h], weight_error)
            outs[b, at], bounds[b, at] = out, bound
            received[b, h, pos], slack[b, h, pos] = p.sum(0), off.sum(0)
    return outs, bounds, received, slack


def prompt(q, kc, cu, starts, tables, lens, block):
    """(received, bounds) [sequences, kv_heads, capacity] of packed causal rows."""
    heads, dim = q.shape[1:]
    kv = kc.shape[2]
    group, capacity = heads // kv, tables.shape[1] * block
    received, slack = torch.zeros(2, len(starts), kv, capacity, dtype=torch.float64, device=kc.device)
    for s in range(len(starts)):
        n, start = int(lens[s]), int(starts[s])
        rows = q[int(cu[s]):int(cu[s + 1])].double()
        rows = rows[:max(0, n - start)]
        if not 0 <= start < n <= capacity or not len(rows):
            continue
        k, pos = rows_of(kc, tables[s], n)
        hidden = pos > start + torch.arange(len(rows), device=kc.device)[:, None]
        for h in range(heads):
            scores = rows[:, h] @ k[:, h // group].T / math.sqrt(dim)
            p = torch.softmax(scores.masked_fill(hidden, float("-inf")), -1)
            p = torch.where(hidden.all(-1, keepdim=True), 0.0, p)
            size = (rows[:, h].abs() @ k[:, h // group].abs().T / math.sqrt(dim)).amax() if len(pos) else 0.0
            received[s, h // group, pos] += p.sum(0)
            slack[s, h // group, pos] += p.sum(0) * fp32_error(dim, size, n)
        # The rows' fp32 sum, in any order.
        slack[s] += received[s] * 2.0 ** -24 * len(rows) * group
    return received, slack


def evict(weights, lens, keep, first=None, recent=0):
    """Positions that stay: a list for each [layer][sequence][kv head] of weights [layers, batch, kv_heads, S]."""
    chosen = []
    for layer in weights.tolist():
        chosen.append([])
        for b, heads in enumerate(layer):
            n = int(lens[b])
            chosen[-1].append([])
            for w in heads:
                f = min(max(0, int(first[b])) if first is not None else 0, keep)
                r = min(recent, keep - f)
                # (NaN above every number; -0 and +0 are equal to a sort, which is stable.)
                order = sorted(range(f, n - r), key=lambda i: (0, 0.0) if math.isnan(w[i]) else (1, -w[i]))
                at = sorted([*range(f), *order[:keep - f - r], *range(n - r, n)]) if n > keep else list(range(n))
                chosen[-1][-1].append(at)
    return chosen


def assert_within(actual, want, bound):
    """|actual - want| <= the bound of the computation, and half a step of the output's type."""
    got, want, bound = actual.double().cpu(), want.cpu(), bound.cpu()
    rounding = torch.finfo(actual.dtype).eps / 2 * (want.abs() + bound) + torch.finfo(actual.dtype).tiny
    off = (got - want).abs() - (bound + rounding)
    assert bool((off <= 0).all()), f"off by {(got - want).abs().max().item()}, {off.max().item()} over the bound"


def assert_weights(after, before, received, slack):
    """The account after = before + received, in fp32; what received nothing has not changed."""
    capacity = received.shape[-1]
    before, after = before.double().cpu(), after.double().cpu()
    received, slack = received.cpu(), slack.cpu()
    # A sum over a group's heads (at most 64 here) and one addition.
    want = before[..., :capacity] + received
    bound = slack + 2.0 ** -24 * (64 * received + want.abs()) + 1e-37
    off = (after[..., :capacity] - want).abs() - bound
    assert bool((off <= 0).all()), f"off by {(after[..., :capacity] - want).abs().max().item()}, {off.max().item()} over"
    assert torch.equal(after[..., capacity:], before[..., capacity:])


def shared_tables(gen, lens, block, groups=(), extra=3, pad=0):
    """Block tables (-1 behind the last page) of distinct shuffled pages, the whole pages of a group's prefix shared.

    groups: (first, last, prefix) with prefix a multiple of block.
    """
    counts = [max(0, -(-n // block)) for n in lens]
    order = torch.randperm(sum(counts) + extra, generator=gen)
    table = torch.full((len(lens), max(1, *counts) + pad), -1, dtype=torch.int64)
    at = 0
    for i, count in enumerate(counts):
        table[i, :count] = order[at:at + count]
        at += count
    for first, last, prefix in groups:
        for b in range(first, last):
            if lens[b] >= prefix:
                table[b, :prefix // block] = table[first, :prefix // block]
    return table, order.numel()


def caches(gen, pages, block, kv_heads, dim, dtype, tables, lens, poison=True):
    """Key and value caches; what no sequence holds is NaN."""
    key, value = (torch.randn(pages, block, kv_heads, dim, generator=gen).to(dtype) for _ in range(2))
    if poison:
        held = torch.zeros(pages, block, dtype=torch.bool)
        for table, n in zip(tables, lens):
            n = min(max(int(n), 0), len(table) * block)
            pos = torch.arange(n)
            page = table[pos // block]
            there = (page >= 0) & (page < pages)
            held[page[there], pos[there] % block] = True
        key[~held] = float("nan")
        value[~held] = float("nan")
    return key, value
