"""The packed 4-bit cache in plain float64 / int64 torch on the CPU: the
rounding rule, the record layout, attention, and the error bounds that the
kernels' tests use."""

from __future__ import annotations

import math

import torch

MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def record_bytes(block, dim):
    return (block * dim // 2 + block * dim // 32 + 15) // 16 * 16


def quantise(rows):
    """Codes [..., dim] and scale bytes [..., dim / 32] of fp16 / bf16 rows, by distance to the eight magnitudes."""
    x = rows.double().unflatten(-1, (-1, 32))
    largest = x.abs().amax(-1)  # NaN where there is one
    byte = torch.full(largest.shape, 104, dtype=torch.int64)
    for e in range(-23, 13):
        byte[largest > 7 * 2.0 ** e] = e + 1 + 127
    byte[largest.isnan()] = 255
    y = (x / torch.exp2(byte.clamp(max=140).double() - 127).unsqueeze(-1)).nan_to_num(0.0, posinf=100.0, neginf=-100.0)
    distance = (y.abs().clamp(max=6.0).unsqueeze(-1) - MAGNITUDES).abs()
    nearest = distance.amin(-1, keepdim=True)
    tied = distance == nearest
    even = tied & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.int().argmax(-1), tied.int().argmax(-1))
    code = code + 8 * torch.signbit(x).long()
    code[byte == 255] = 0
    return code.flatten(-2), byte


def values(code, byte):
    """float64 values of codes [..., dim] and scale bytes [..., dim / 32]."""
    scale = torch.where(byte == 255, torch.nan, torch.exp2(byte.double() - 127))
    signed = torch.cat((MAGNITUDES, -MAGNITUDES))[code]
    return (signed.unflatten(-1, (-1, 32)) * scale.unsqueeze(-1)).flatten(-2)


def split(cache, block, dim):
    """Codes [pages, kv_heads, block, dim] and scale bytes of a packed cache on the CPU."""
    c = cache.long()
    codes = c[..., :block * dim // 2].unflatten(-1, (block, dim // 2))
    code = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
    return code, c[..., block * dim // 2:block * dim // 2 + block * dim // 32].unflatten(-1, (block, dim // 32))


def join(code, byte):
    """The packed cache of codes [pages, kv_heads, block, dim] and scale bytes; its padding is zeros."""
    pages, heads, block, dim = code.shape
    packed = (code[..., 0::2] + 16 * code[..., 1::2]).reshape(pages, heads, -1)
    cache = torch.zeros(pages, heads, record_bytes(block, dim), dtype=torch.int64)
    cache[..., :packed.shape[-1]] = packed
    cache[..., packed.shape[-1]:packed.shape[-1] + block * dim // 32] = byte.reshape(pages, heads, -1)
    return cache.to(torch.uint8)


def packed(rows):
    """The packed cache of rows [pages, kv_heads, block, dim]."""
    return join(*quantise(rows))


def cache_values(cache, block, dim):
    """float64 [pages, block, kv_heads, dim]."""
    return values(*split(cache, block, dim)).transpose(1, 2)


def random_caches(gen, pages, heads, block, dim, dtype):
    return [packed(torch.randn(pages, heads, block, dim, generator=gen).to(dtype)) for _ in range(2)]


def attention(query, key, value):
    """One row: query [dim], key / value [n, dim] in float64 -> (output, error bound without the output's rounding).

    Every probability is rounded to fp16 (half a step: 2^-11 of it); a score
    is a sum of dim products in fp32 (and the exponential of an fp32 value),
    the sums over n keys are fp32 sums.
    """
    n, dim = key.shape
    if n == 0:
        zero = torch.zeros(dim, dtype=torch.float64)
        return zero, zero
    scores = key @ query / math.sqrt(dim)
    weights = torch.softmax(scores, 0)
    out = weights @ value
    size = (key.abs() @ query.abs() / math.sqrt(dim)).max().item()
    spread = weights @ value.abs()
    return out, spread * (2.0 ** -11 + 2.0 ** -23 * (2 * (dim + 8) * (size + 1) + n + 64))


def decode_oracle(query, kc, vc, tables, lens, block):
    """(outputs, bounds), float64 [batch, heads, dim]; absent pages are skipped."""
    batch, heads, dim = query.shape
    keys, vals = cache_values(kc, block, dim), cache_values(vc, block, dim)
    pages, _, kv, _ = keys.shape
    outs, bounds = torch.zeros(2, batch, heads, dim, dtype=torch.float64)
    for b in range(batch):
        n = int(lens[b])
        if not 0 < n <= tables.shape[1] * block:
            continue
        pos = torch.arange(n)
        page = tables[b][pos // block]
        pos, page = pos[(page >= 0) & (page < pages)], page[(page >= 0) & (page < pages)]
        k, v = keys[page, pos % block], vals[page, pos % block]
        for h in range(heads):
            outs[b, h], bounds[b, h] = attention(query[b, h].double(), k[:, h // (heads // kv)],
                                                 v[:, h // (heads // kv)])
    return outs, bounds


def prefill_oracle(query, kc, vc, cu, starts, tables, lens, block):
    """(outputs, bounds), float64 [tokens, heads, dim]; rows that no sequence owns or that see no key are zeros."""
    tokens, heads, dim = query.shape
    keys, vals = cache_values(kc, block, dim), cache_values(vc, block, dim)
    pages, _, kv, _ = keys.shape
    outs, bounds = torch.zeros(2, tokens, heads, dim, dtype=torch.float64)
    for s in range(len(starts)):
        n, start = int(lens[s]), int(starts[s])
        if not (0 <= start < n <= tables.shape[1] * block):
            continue
        pos = torch.arange(n)
        page = tables[s][pos // block]
        pos, page = pos[(page >= 0) & (page < pages)], page[(page >= 0) & (page < pages)]
        k, v = keys[page, pos % block], vals[page, pos % block]
        for t in range(int(cu[s]), int(cu[s + 1])):
            at = start + t - int(cu[s])
            if at >= n:
                continue
            seen = pos <= at
            for h in range(heads):
                outs[t, h], bounds[t, h] = attention(query[t, h].double(), k[seen][:, h // (heads // kv)],
                                                     v[seen][:, h // (heads // kv)])
    return outs, bounds


def assert_within(actual, want, bound):
    """|actual - want| <= half a step of the output's type, and the bound of the computation."""
    got = actual.double().cpu()
    rounding = torch.finfo(actual.dtype).eps / 2 * (want.abs() + bound) + torch.finfo(actual.dtype).tiny
    off = (got - want).abs() - (bound + rounding)
    assert bool((off <= 0).all()), f"off by {(got - want).abs().max().item()}, {off.max().item()} over the bound"


def tables_of(gen, lens, block, extra=3, pad=0):
    """Distinct shuffled pages for each length (-1 past its last page), and the number of pages."""
    counts = [max(0, -(-n // block)) for n in lens]
    order = torch.randperm(sum(counts) + extra, generator=gen)
    table = torch.full((len(lens), max(1, *counts) + pad), -1, dtype=torch.int64)
    at = 0
    for i, count in enumerate(counts):
        table[i, :count] = order[at:at + count]
        at += count
    return table, order.numel()
