"""Timing cases of the 4-bit KV cache and of the cache's page operators.

A serving engine that holds its paged K/V cache in 4 bits writes every new
row through a quantiser, attends over the packed pages in its decode steps
and prompt chunks, and reads rows back where another path wants them in 16
bits.  Beam search and parallel sampling fork requests, which copies the page
a request is still writing; a fragmented pool is compacted by moving pages
and renumbering the block tables.

A packed cache of one layer is uint8 ``[pages, kv_heads, record]``.  A record
holds ``block`` tokens of one kv head: first ``block * dim / 2`` bytes of
codes (token-major; the low four bits of a byte are the even dim), then
``block * dim / 32`` scale bytes, then zeros up to a multiple of 16.  A code
is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; 32 dims share the power of
two 2^(byte - 127), the smallest one in [2^-23, 2^13] whose 7 covers the
largest magnitude.

Sizes follow the package's workloads (16 query / 8 kv heads of 128, pages of
16 or 256 tokens, 28 layers) and its tests (groups of 1 to 8 heads, other
head dims and page sizes, odd lengths).
"""

import functools
import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


@functools.lru_cache(maxsize=1)
def _package():
    """The framework's entry points (only where `own` is true)."""
    sys.path.insert(0, os.path.join(os.getcwd(), "myvllm-mini-engine_amd"))
    from mini_engine_hip.kernels import fp4, pages

    return fp4, pages


# ---------------------------------------------------------------------------
# The cases.
# ---------------------------------------------------------------------------
def _store(name, **kw):
    return {"name": name, "kind": "store", "tokens": 32, "kv_heads": 8, "dim": 128, "block": 16, "dtype": "bf16", **kw}


def _decode(name, **kw):
    case = {"kind": "decode", "batch": 1, "context": 128, "ragged": False, "heads": 16, "kv_heads": 8, "dim": 128,
            "block": 256, "dtype": "fp16", "mix": 1}
    return {"name": name, **case, **kw}


def _prefill(name, **kw):
    case = {"kind": "prefill", "seqs": 8, "new": 128, "prior": 3968, "ragged": False, "heads": 16, "kv_heads": 8,
            "dim": 128, "block": 256, "dtype": "bf16", "mix": 1}
    return {"name": name, **case, **kw}


def _pages(name, kind, **kw):
    case = {"kind": kind, "layers": 28, "pages": 512, "moves": 8, "kv_heads": 8, "dim": 128, "block": 16,
            "format": "fp4", "batch": 32, "width": 32, "mix": 1}
    return {"name": name, **case, **kw}


def listed():
    return [
        # One decode step's new rows of a batch of 32: all latency.
        _store("store_b32"),
        # The rows of a large prompt batch.
        _store("store_16384", tokens=16384, block=256, dtype="fp16"),
        # One request, a short context: the interactive step.
        _decode("decode4_b1_ctx128"),
        # A server's mixed batch on small pages.
        _decode("decode4_ragged_b64", batch=64, context=4096, ragged=True, block=16, dtype="bf16"),
        # A few very long contexts, eight query heads to a kv head: what four bits are held for.
        _decode("decode4_group8_b4_65536", batch=4, context=65536, heads=32, kv_heads=4, dtype="bf16"),
        # A chunked-prefill batch on top of cached context.
        _prefill("prefill4_8x128"),
        # Prompts of many lengths admitted together on small pages, seven query heads to a kv head.
        _prefill("prefill4_mixed_12", seqs=12, new=500, prior=700, ragged=True, heads=28, kv_heads=4, block=16,
                 dtype="fp16"),
        # Long prompts without cached context.
        _prefill("prefill4_2x4096", seqs=2, new=4096, prior=0),
        # Eight requests fork: the page each is writing is copied in every layer.
        _pages("fork_8_pages", "copy"),
        # Copies of whole long prefixes, 16-bit cache.
        _pages("copy_512_pages_bf16", "copy", format="bf16", pages=1100, moves=512),
        # A light compaction of a packed pool between two steps.
        _pages("compact_24_of_512", "compact", moves=24),
        # A pool of large 16-bit pages pulled together.
        _pages("compact_16_large_pages", "compact", format="bf16", pages=64, moves=16, block=256, batch=8, width=8),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: the kind, then heads, type and page size, then sizes
    spread over the logarithm of their range; odd ones are the rule."""
    kind = rng.choice(["store", "decode", "decode", "decode", "prefill", "prefill", "copy", "compact"])
    heads, kv_heads, dim = rng.choice([(16, 8, 128), (16, 8, 128), (32, 8, 128), (28, 4, 128), (32, 4, 128),
                                       (8, 8, 128), (40, 8, 128), (16, 1, 128), (14, 2, 64), (16, 8, 64), (12, 4, 96),
                                       (8, 2, 256), (4, 4, 32)])
    block = rng.choice([16, 16, 256, 256, 32, 7])
    dtype = rng.choice(["fp16", "bf16"])
    mix = rng.randrange(1 << 30)
    if kind == "store":
        return {"kind": kind, "tokens": _log_int(rng, 1, 16384), "kv_heads": kv_heads, "dim": dim, "block": block,
                "dtype": dtype, "mix": mix}
    if kind == "decode":
        # At most as many cached values as the long case has.
        room = 4 * 65536 * 4 * 128 // (kv_heads * dim)
        batch = _log_int(rng, 1, 128)
        return {"kind": kind, "batch": batch, "context": _log_int(rng, 1, min(131072, room // batch)),
                "ragged": rng.random() < 0.6, "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block,
                "dtype": dtype, "mix": mix}
    if kind == "prefill":
        seqs = _log_int(rng, 1, 24)
        new = _log_int(rng, 1, 4096 // max(1, seqs // 2))
        # At most as many products as the long case has: 2 x 4096 x 4096 / 2 pairs, 16 heads of 128.
        room = 4096 * 4096 * 16 * 128 // (heads * dim)
        new = max(1, min(new, int(math.sqrt(2 * room / seqs))))
        left = (room - seqs * new * new // 2) // (seqs * new) + 1
        prior = rng.choice([0, _log_int(rng, 1, max(2, min(16384, left)))])
        return {"kind": kind, "seqs": seqs, "new": new, "prior": prior, "ragged": rng.random() < 0.6, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "block": block, "dtype": dtype, "mix": mix}
    form = rng.choice(["fp4", "bf16", "fp16"])
    layers = _log_int(rng, 1, 36)
    case = {"kind": kind, "layers": layers, "kv_heads": kv_heads, "dim": dim, "block": block, "format": form,
            "mix": mix}
    page = 2 * layers * _page_bytes(case)
    pages = max(8, min(_log_int(rng, 16, 4096), 2 * 28 * 1100 * 2 * 16 * 8 * 128 // page))
    most = max(1, min(pages // 2, 2 * 28 * 512 * 2 * 16 * 8 * 128 // page))
    batch = _log_int(rng, 1, 64)
    return {**case, "pages": pages, "moves": _log_int(rng, 1, most), "batch": batch,
            "width": max(1, (pages - most) // batch)}


# ---------------------------------------------------------------------------
# Lengths, tables and sizes: plain values of the case.
# ---------------------------------------------------------------------------
def _record(block, dim):
    return -(-(block * (dim // 2 + dim // 32)) // 16) * 16


def _page_bytes(case):
    """Bytes of one page of one layer's keys (or values)."""
    if case["format"] == "fp4":
        return case["kv_heads"] * _record(case["block"], case["dim"])
    return 2 * case["block"] * case["kv_heads"] * case["dim"]


def _lengths(count, top, ragged, mix, low=1):
    if not ragged:
        return [top] * count
    rng = random.Random(mix)
    return [rng.randint(low, max(low, top)) for _ in range(count)]


def _contexts(case):
    return _lengths(case["batch"], case["context"], case["ragged"], case["mix"])


def _chunks(case):
    """(new tokens, prior tokens) of each sequence of a prefill batch; priors always vary."""
    new = _lengths(case["seqs"], case["new"], case["ragged"], case["mix"], low=max(1, case["new"] // 16))
    return new, _lengths(case["seqs"], case["prior"], True, case["mix"] + 1, low=0)


def _tables(lens, block, seed):
    """Block tables of shuffled distinct pages, -1 past a sequence's last."""
    pages = [math.ceil(n / block) for n in lens]
    order = list(range(sum(pages) + 7))
    random.Random(seed).shuffle(order)
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int64)
    at = 0
    for i, count in enumerate(pages):
        table[i, :count] = torch.tensor(order[at:at + count], dtype=torch.int64)
        at += count
    return table, len(order)


# ---------------------------------------------------------------------------
# The packed format, in elementary operations.
# ---------------------------------------------------------------------------
def _quantise(x):
    """(codes [..., dim / 2], scale bytes [..., dim / 32]), uint8, of rows x in 16 bits."""
    blocks = x.float().unflatten(-1, (-1, 32))
    mantissa, exponent = torch.frexp(blocks.abs().amax(-1))
    # The largest magnitude is mantissa * 2^exponent, mantissa in [0.5, 1): 8 mantissa <= 7 fits 2^(exponent - 3).
    power = (exponent - 3 + (mantissa > 0.875)).clamp(-23, 13)
    scaled = torch.ldexp(blocks, -power.unsqueeze(-1))
    a = scaled.abs()
    # To the nearest, ties to the even code.
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * (scaled < 0)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], (power + 127).to(torch.uint8)


def _views(cache, block, dim):
    """The codes [pages, kv_heads, block, dim / 2] and scales [pages, kv_heads, block, dim / 32] of a packed cache."""
    codes = block * dim // 2
    return (cache[..., :codes].unflatten(-1, (block, dim // 2)),
            cache[..., codes:codes + block * dim // 32].unflatten(-1, (block, dim // 32)))


def _values(codes, scales):
    """The 32-bit values of codes [..., dim / 2] and scale bytes [..., dim / 32]."""
    table = torch.tensor(MAGNITUDES + [-v for v in MAGNITUDES], device=codes.device)
    nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    powers = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    return (table[nibbles.int()].unflatten(-1, (-1, 32)) * powers.unsqueeze(-1)).flatten(-2)


def _gathered(cache, tables, block, dim):
    """Values [sequences, kv_heads, table width * block, dim] of every table's pages."""
    codes, scales = _views(cache[tables.clamp(min=0)], block, dim)  # [S, W, Hkv, block, .]
    return _values(codes, scales).permute(0, 2, 1, 3, 4).flatten(2, 3)


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _rows(gen, dtype, tokens, kv_heads, dim):
    """K and V rows: the channels of keys differ in size, as after a trained projection."""
    channel = torch.exp(0.5 * _randn(gen, kv_heads, dim))
    return (_randn(gen, tokens, kv_heads, dim) * channel).to(dtype), _randn(gen, tokens, kv_heads, dim).to(dtype)


def _packed(gen, dtype, pages, kv_heads, block, dim):
    """A layer's packed key and value caches, full of rows."""
    caches = []
    for rows in _rows(gen, dtype, pages * block, kv_heads, dim):
        cache = torch.zeros(pages, kv_heads, _record(block, dim), dtype=torch.uint8, device=DEVICE)
        codes, scales = _quantise(rows.unflatten(0, (pages, block)).transpose(1, 2))
        for view, part in zip(_views(cache, block, dim), (codes, scales)):
            view.copy_(part)
        caches.append(cache)
    return caches


def _prepare_store(case, gen, seed):
    block, tokens = case["block"], case["tokens"]
    pages = math.ceil(tokens / block) + 7
    shape = (pages, case["kv_heads"], _record(block, case["dim"]))
    # Consecutive positions of pages in shuffled order.
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed)))
    pos = torch.arange(tokens)
    key, value = _rows(gen, DTYPES[case["dtype"]], tokens, case["kv_heads"], case["dim"])
    return {"key_cache": torch.zeros(shape, dtype=torch.uint8, device=DEVICE),
            "value_cache": torch.zeros(shape, dtype=torch.uint8, device=DEVICE),
            "slots": (order[pos // block] * block + pos % block).to(DEVICE), "key": key, "value": value}


def _prepare_decode(case, gen, seed):
    lens = _contexts(case)
    table, pages = _tables(lens, case["block"], seed)
    dtype = DTYPES[case["dtype"]]
    kc, vc = _packed(gen, dtype, pages, case["kv_heads"], case["block"], case["dim"])
    query = _randn(gen, case["batch"], case["heads"], case["dim"]).to(dtype)
    return {"query": query, "key_cache": kc, "value_cache": vc, "tables": table.to(DEVICE),
            "lens": torch.tensor(lens, device=DEVICE)}


def _prepare_prefill(case, gen, seed):
    new, prior = _chunks(case)
    lens = [n + p for n, p in zip(new, prior)]
    table, pages = _tables(lens, case["block"], seed)
    dtype = DTYPES[case["dtype"]]
    kc, vc = _packed(gen, dtype, pages, case["kv_heads"], case["block"], case["dim"])
    query = _randn(gen, sum(new), case["heads"], case["dim"]).to(dtype)
    cu = torch.tensor([0] + new).cumsum(0)
    return {"query": query, "key_cache": kc, "value_cache": vc, "tables": table.to(DEVICE), "cu": cu.to(DEVICE),
            "starts": torch.tensor(prior, device=DEVICE), "lens": torch.tensor(lens, device=DEVICE),
            "longest": max(new)}


def _prepare_pages(case, gen, seed):
    layers, pages, moves = case["layers"], case["pages"], case["moves"]
    if case["format"] == "fp4":
        planes = torch.randint(0, 256, (2, layers, pages, case["kv_heads"], _record(case["block"], case["dim"])),
                               generator=gen, device=DEVICE, dtype=torch.uint8)
    else:
        planes = torch.empty((2, layers, pages, case["block"], case["kv_heads"], case["dim"]),
                             dtype=DTYPES[case["format"]], device=DEVICE).normal_(generator=gen)
    rng = random.Random(int(seed))
    order = list(range(pages))
    rng.shuffle(order)
    if case["kind"] == "copy":
        src, dst = order[:moves], order[moves:2 * moves]
    else:  # live pages above the holes that they move into
        src, dst = sorted(range(pages - moves, pages)), sorted(rng.sample(range(pages - moves), moves))
    holes = set(dst)
    live = [p for p in order if p not in holes]
    table = torch.full((case["batch"], case["width"]), -1, dtype=torch.int64)
    for b in range(case["batch"]):  # requests of many lengths; prefix pages are shared
        count = rng.randint(1, case["width"])
        at = rng.randrange(len(live))
        table[b, :count] = torch.tensor([live[(at + i) % len(live)] for i in range(count)])
    return {"planes": planes, "src": torch.tensor(src, device=DEVICE), "dst": torch.tensor(dst, device=DEVICE),
            "tables": table.to(DEVICE)}


def prepare(case, seed):
    make = {"store": _prepare_store, "decode": _prepare_decode, "prefill": _prepare_prefill, "copy": _prepare_pages,
            "compact": _prepare_pages}[case["kind"]]
    return {"case": case, **make(case, _generator(seed), seed)}


# ---------------------------------------------------------------------------
# run
# ---------------------------------------------------------------------------
def _store_plain(state, block, dim):
    page, offset = state["slots"] // block, state["slots"] % block
    read = []
    for cache, rows in ((state["key_cache"], state["key"]), (state["value_cache"], state["value"])):
        codes, scales = _views(cache, block, dim)
        codes[page, :, offset], scales[page, :, offset] = _quantise(rows)
        read.append(_values(codes[page, :, offset], scales[page, :, offset]).to(rows.dtype))
    return read


def _run_store(state, case):
    block, dim = case["block"], case["dim"]
    if own:
        fp4, _ = _package()
        fp4.write_kv_cache_slots_fp4(state["key_cache"], state["value_cache"], state["slots"], state["key"],
                                     state["value"], block, validate=False)
        return fp4.gather_kv_cache_slots_fp4(state["key_cache"], state["value_cache"], state["slots"], block, dim,
                                             state["key"].dtype, validate=False)
    return _store_plain(state, block, dim)


def _decode_plain(state, block, dim):
    query, lens = state["query"], state["lens"]
    key = _gathered(state["key_cache"], state["tables"], block, dim)  # [B, Hkv, N, D]
    grouped = query.float().unflatten(1, (key.shape[1], -1))  # [B, Hkv, G, D]
    scores = grouped @ key.transpose(-1, -2) / math.sqrt(dim)
    del key
    scores.masked_fill_(torch.arange(scores.shape[-1], device=DEVICE) >= lens[:, None, None, None], float("-inf"))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights /= weights.sum(-1, keepdim=True)
    out = weights @ _gathered(state["value_cache"], state["tables"], block, dim)
    return out.flatten(1, 2).to(query.dtype)


def _run_decode(state, case):
    if own:
        fp4, _ = _package()
        return fp4.paged_attention_fp4(state["query"], state["key_cache"], state["value_cache"], state["tables"],
                                       state["lens"], case["block"], validate=False)
    return _decode_plain(state, case["block"], case["dim"])


def _prefill_plain(state, block, dim):
    query, cu, starts = state["query"], state["cu"], state["starts"]
    rows = torch.arange(query.shape[0], device=DEVICE)
    seq = torch.searchsorted(cu, rows, right=True) - 1
    local = rows - cu[seq]
    padded = torch.zeros(starts.shape[0], state["longest"], *query.shape[1:], device=DEVICE)  # [S, T, H, D]
    padded[seq, local] = query.float()
    key = _gathered(state["key_cache"], state["tables"], block, dim)  # [S, Hkv, N, D]
    grouped = padded.permute(0, 2, 1, 3).unflatten(1, (key.shape[1], -1))  # [S, Hkv, G, T, D]
    scores = grouped.flatten(2, 3) @ key.transpose(-1, -2) / math.sqrt(dim)
    del key
    scores = scores.unflatten(2, grouped.shape[2:4])  # [S, Hkv, G, T, N]
    last = starts[:, None] + torch.arange(scores.shape[3], device=DEVICE)  # [S, T]
    hidden = torch.arange(scores.shape[-1], device=DEVICE) > last[:, :, None]  # [S, T, N]
    scores.masked_fill_(hidden[:, None, None], float("-inf"))
    scores -= scores.amax(-1, keepdim=True)
    weights = scores.exp_()
    weights /= weights.sum(-1, keepdim=True)
    out = weights.flatten(2, 3) @ _gathered(state["value_cache"], state["tables"], block, dim)
    out = out.unflatten(2, grouped.shape[2:4]).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [S, T, H, D]
    return out[seq, local].to(query.dtype)


def _run_prefill(state, case):
    if own:
        fp4, _ = _package()
        return fp4.paged_prefill_attention_fp4(state["query"], state["key_cache"], state["value_cache"], state["cu"],
                                               state["starts"], state["tables"], state["lens"], case["block"],
                                               validate=False)
    return _prefill_plain(state, case["block"], case["dim"])


def _run_copy(state, case):
    if own:
        _, pages = _package()
        pages.copy_kv_pages(state["planes"], state["src"], state["dst"], page_dim=2, validate=False)
    else:
        state["planes"][:, :, state["dst"]] = state["planes"][:, :, state["src"]]
    return state["planes"]


def _run_compact(state, case):
    if own:
        _, pages = _package()
        pages.compact_kv_pages(state["planes"], state["src"], state["dst"], state["tables"], page_dim=2, validate=False)
    else:
        planes, tables = state["planes"], state["tables"]
        planes[:, :, state["dst"]] = planes[:, :, state["src"]]
        number = torch.arange(planes.shape[2], device=DEVICE)
        number[state["src"]] = state["dst"]
        tables.copy_(torch.where(tables >= 0, number[tables.clamp(min=0)], tables))
    return [state["planes"], state["tables"]]


_RUN = {"store": _run_store, "decode": _run_decode, "prefill": _run_prefill, "copy": _run_copy, "compact": _run_compact}


def run(state):
    return _RUN[state["case"]["kind"]](state, state["case"])


# ---------------------------------------------------------------------------
# work and exact
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind in ("copy", "compact"):
        moved = 2 * case["layers"] * case["moves"] * _page_bytes(case)
        table = 16 * case["batch"] * case["width"] if kind == "compact" else 0
        return {"bytes": 2 * moved + 16 * case["moves"] + table, "flops": 0}
    token = 2 * case["kv_heads"] * (case["dim"] // 2 + case["dim"] // 32)  # packed K and V
    if kind == "store":
        rows = 4 * case["kv_heads"] * case["dim"]  # K and V in 16 bits, in and out
        return {"bytes": case["tokens"] * (2 * rows + token + 8), "flops": 0}
    width = case["heads"] * case["dim"]
    if kind == "decode":
        total = sum(_contexts(case))
        return {"bytes": total * token + 4 * case["batch"] * width + 8 * math.ceil(total / case["block"]),
                "flops": 4 * width * total}
    new, prior = _chunks(case)
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, prior))
    total = sum(new) + sum(prior)
    return {"bytes": total * token + 4 * sum(new) * width, "flops": 4 * width * pairs}


def _exact_rows(x):
    """What rows in 16 bits become in the packed format, in 64 bits: the nearest multiple of the step that each
    magnitude's binade has."""
    blocks = x.double().unflatten(-1, (-1, 32))
    largest = blocks.abs().amax(-1, keepdim=True)
    unit = torch.full_like(largest, 2.0 ** -23)
    for power in range(-23, 13):
        unit = torch.where(largest > 7 * unit, 2.0 * unit, unit)
    y = blocks / unit
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    return (torch.round(y / step) * step).clamp(-6, 6).mul(unit).flatten(-2)  # round() takes ties to even


def _exact_cache(cache, pages, tokens, block, dim):
    """The first `tokens` rows of a page list, [kv_heads, tokens, dim] in 64 bits."""
    record = cache[pages].to(torch.int64)  # [P, Hkv, R]
    codes = record[..., :block * dim // 2].reshape(*record.shape[:2], block, dim // 2)
    scales = record[..., block * dim // 2:block * dim // 2 + block * dim // 32].reshape(*record.shape[:2], block, -1)
    nibbles = torch.stack((codes % 16, codes // 16), -1).reshape(*codes.shape[:3], dim)
    exponent, half = (nibbles % 8) // 2, (nibbles % 2).double()
    value = torch.where(exponent == 0, 0.5 * half, (1 + 0.5 * half) * 2.0 ** (exponent - 1).double())
    value = torch.where(nibbles >= 8, -value, value) * (2.0 ** (scales - 127).double()).repeat_interleave(32, -1)
    return value.permute(1, 0, 2, 3).reshape(record.shape[1], -1, dim)[:, :tokens]


def _exact_attention(query, key, value, first):
    """query [n, heads, dim] at positions first.. over key / value [kv_heads, tokens, dim], causal, in 64 bits."""
    n, heads, dim = query.shape
    group = heads // key.shape[0]
    out = torch.empty(n, heads, dim, dtype=torch.float64, device=query.device)
    visible = torch.arange(key.shape[1], device=query.device) <= first + torch.arange(n, device=query.device)[:, None]
    for h in range(heads):
        scores = query[:, h].double() @ key[h // group].T * dim ** -0.5
        out[:, h] = torch.softmax(scores.masked_fill(~visible, float("-inf")), -1) @ value[h // group]
    return out


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind in ("copy", "compact"):
        planes, src, dst = state["planes"], state["src"].tolist(), state["dst"].tolist()
        moved = planes.clone() if planes.dtype == torch.uint8 else planes.double()
        for s, d in zip(src, dst):
            moved[:, :, d] = planes[:, :, s].to(moved.dtype)
        if kind == "copy":
            return moved
        number = dict(zip(src, dst))
        return [moved, torch.tensor([[number.get(p, p) for p in row] for row in state["tables"].tolist()])]
    if kind == "store":
        return [_exact_rows(state["key"]), _exact_rows(state["value"])]
    block, dim = case["block"], case["dim"]
    if kind == "decode":
        new, prior = [1] * case["batch"], [n - 1 for n in _contexts(case)]
    else:
        new, prior = _chunks(case)
    outs, at = [], 0
    for i, (n, p) in enumerate(zip(new, prior)):
        pages = state["tables"][i, :math.ceil((n + p) / block)]
        rows = [_exact_cache(state[name], pages, n + p, block, dim) for name in ("key_cache", "value_cache")]
        outs.append(_exact_attention(state["query"][at:at + n], *rows, p))
        at += n
    return torch.cat(outs)
