"""Writing rows into the packed 4-bit cache and reading them back, on the GPU,
against the rule in float64 (bit for bit)."""

import pytest
import torch

import fp4_cases as f4
from mini_engine_hip.kernels.fp4 import (fp4_record_bytes, gather_kv_cache_fp4, gather_kv_cache_slots_fp4,
                                         write_kv_cache_batch_fp4, write_kv_cache_slots_fp4)

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def caches(pages, heads, block, dim, fill=0xA5):
    return [torch.full((pages, heads, fp4_record_bytes(block, dim)), fill, dtype=torch.uint8, device=DEV)
            for _ in range(2)]


def written(before, rows, slots, block):
    """The cache after rows [tokens, heads, dim] went to their slots."""
    dim = rows.shape[-1]
    code, byte = f4.split(before.cpu(), block, dim)
    new_code, new_byte = f4.quantise(rows.cpu())
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < before.shape[0] * block:
            code[slot // block, :, slot % block] = new_code[t]
            byte[slot // block, :, slot % block] = new_byte[t]
    after = f4.join(code, byte)
    used = block * (dim // 2 + dim // 32)
    after[..., used:] = before.cpu()[..., used:]  # the padding is nobody's
    return after


def patterns(dtype):
    """Every 16-bit pattern, in blocks of neighbours, of random company, and alone beside the block's largest."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    gen = torch.Generator().manual_seed(1)
    mixed = every[torch.randperm(65536, generator=gen)]
    mixed = mixed[torch.isfinite(mixed)]
    mixed = mixed[:mixed.numel() // 32 * 32]
    tops = torch.tensor([2.0 ** -24, 2.0 ** -20, 3.0e-5, 1.75, 1.7578125, 7.0, 100.0, 50000.0]).to(dtype)
    alone = []
    for top in tops:  # every smaller pattern beside the top of its block
        smaller = every[every.abs() <= top]
        smaller = smaller[:smaller.numel() // 31 * 31].view(-1, 31)
        alone.append(torch.cat((top.expand(smaller.shape[0], 1), smaller), 1).flatten())
    alone = torch.cat(alone)
    return torch.cat((every, mixed, alone)).view(-1, 32)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_pattern_is_rounded_by_the_rule(dtype):
    """All 16-bit values, infinities and NaNs among them, key and value alike."""
    rows = patterns(dtype)
    rows = rows[:rows.shape[0] // 8 * 8].view(-1, 2, 128)  # [tokens, 2 heads, 128]
    tokens, block = rows.shape[0], 16
    pages = -(-tokens // block)
    kc, vc = caches(pages, 2, block, 128)
    slots = torch.arange(tokens)
    before = kc.clone()
    write_kv_cache_slots_fp4(kc, vc, slots.to(DEV), rows.to(DEV), rows.flip(0).to(DEV), block)
    assert torch.equal(kc.cpu(), written(before, rows, slots, block))
    assert torch.equal(vc.cpu(), written(before, rows.flip(0), slots, block))
    k, v = gather_kv_cache_slots_fp4(kc, vc, slots.to(DEV), block, 128, dtype)
    want = f4.values(*f4.quantise(rows))
    assert torch.equal(k.cpu().double().nan_to_num(1e9), want.nan_to_num(1e9))
    assert torch.equal(v.cpu().double().nan_to_num(1e9), want.flip(0).nan_to_num(1e9))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("block,heads", [(1, 1), (7, 3), (16, 8), (256, 2)])
def test_write_and_read_back(dtype, dim, block, heads):
    gen = torch.Generator().manual_seed(dim + block)
    tokens, pages = 37, 40 // block + 3
    key, value = (torch.randn(tokens, heads, dim, generator=gen).to(dtype) for _ in range(2))
    slots = torch.randperm(pages * block, generator=gen)[:tokens]
    kc, vc = caches(pages, heads, block, dim)
    before = kc.clone()
    write_kv_cache_slots_fp4(kc, vc, slots.to(DEV), key.to(DEV), value.to(DEV), block)
    assert torch.equal(kc.cpu(), written(before, key, slots, block))
    assert torch.equal(vc.cpu(), written(before, value, slots, block))
    for out in TYPES:  # both types hold every value of the format
        k, v = gather_kv_cache_slots_fp4(kc, vc, slots.to(DEV), block, dim, out)
        assert torch.equal(k.cpu().double(), f4.values(*f4.quantise(key)))
        assert torch.equal(v.cpu().double(), f4.values(*f4.quantise(value)))


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_more_rows_than_the_chip_takes_at_once(dtype, strided):
    """Lanes with two pieces, the last ones with one; slots that do not exist among them."""
    gen = torch.Generator().manual_seed(8)
    tokens, heads, dim, block, pages = 769, 57, 96, 7, 120
    key, value = (torch.randn(tokens, heads, dim, generator=gen).to(dtype) for _ in range(2))
    slots = torch.randperm(pages * block, generator=gen)[:tokens]
    slots[5::50] = -1
    slots[9::50] = pages * block + 3
    exists = (slots >= 0) & (slots < pages * block)
    sources = [x.to(DEV) for x in (key, value)]
    if strided:  # rows that start at odd places
        sources = [torch.nn.functional.pad(x.view(tokens, -1), (1, 0))[:, 1:].view(tokens, heads, dim) for x in sources]
    kc, vc = caches(pages, heads, block, dim)
    before = kc.clone()
    write_kv_cache_slots_fp4(kc, vc, slots.to(DEV), *sources, block, validate=False)
    assert torch.equal(kc.cpu(), written(before, key, slots, block))
    assert torch.equal(vc.cpu(), written(before, value, slots, block))
    k, v = gather_kv_cache_slots_fp4(kc, vc, slots.to(DEV), block, dim, dtype, validate=False)
    for got, rows in ((k, key), (v, value)):
        assert torch.equal(got.cpu().double(), f4.values(*f4.quantise(rows)) * exists.view(-1, 1, 1))
    tables = torch.arange(pages, device=DEV).view(1, pages).expand(tokens, pages).contiguous()
    again = caches(pages, heads, block, dim)
    write_kv_cache_batch_fp4(*again, tables, slots.to(DEV), *sources, block, validate=False)
    assert torch.equal(again[0], kc) and torch.equal(again[1], vc)
    k, _ = gather_kv_cache_fp4(kc, vc, tables[0].contiguous(), pages * block, block, dim, dtype)
    # (Slots that nothing wrote hold the fill, whose scale 2^38 no written block has: past 65504 fp16 reads infinity.)
    assert torch.equal(k.cpu(), f4.cache_values(kc.cpu(), block, dim).flatten(0, 1).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_unaligned_rows(dtype):
    """Slices of a fused projection, an odd token stride, rows that start two bytes off, and a view that is copied."""
    gen = torch.Generator().manual_seed(3)
    tokens, heads, dim, block = 19, 4, 64, 16
    slots = torch.randperm(48, generator=gen)[:tokens].to(DEV)
    fused = torch.randn(tokens, 3 * heads * dim + 1, generator=gen).to(dtype).to(DEV)
    flat = torch.randn(tokens * heads * dim + 1, generator=gen).to(dtype).to(DEV)
    views = [fused[:, 1:1 + heads * dim].unflatten(1, (heads, dim)), flat[1:].view(tokens, heads, dim),
             fused[:, :heads * dim].unflatten(1, (heads, dim)),
             torch.randn(heads, tokens, dim, generator=gen).to(dtype).to(DEV).transpose(0, 1)]
    for key in views:
        for value in views[::-1]:
            kc, vc = caches(3, heads, block, dim)
            before = kc.clone()
            write_kv_cache_slots_fp4(kc, vc, slots, key, value, block)
            assert torch.equal(kc.cpu(), written(before, key, slots.cpu(), block))
            assert torch.equal(vc.cpu(), written(before, value, slots.cpu(), block))


def test_trusted_slots_out_of_range_are_skipped_and_read_as_zeros():
    gen = torch.Generator().manual_seed(4)
    key, value = (torch.randn(6, 2, 32, generator=gen).half() for _ in range(2))
    slots = torch.tensor([5, -1, 1 << 40, 64, 63, -(1 << 62)])
    kc, vc = caches(4, 2, 16, 32)
    before = kc.clone()
    write_kv_cache_slots_fp4(kc, vc, slots.to(DEV), key.to(DEV), value.to(DEV), 16, validate=False)
    assert torch.equal(kc.cpu(), written(before, key, slots, 16))
    assert torch.equal(vc.cpu(), written(before, value, slots, 16))
    k, _ = gather_kv_cache_slots_fp4(kc, vc, slots.to(DEV), 16, 32, torch.float16, validate=False)
    want = f4.values(*f4.quantise(key))
    want[[1, 2, 3, 5]] = 0
    assert torch.equal(k.cpu().double(), want)


def test_decode_step_write_and_page_list_read():
    """One row per sequence through block tables; rows without a place are skipped; a page list read in order."""
    gen = torch.Generator().manual_seed(5)
    heads, dim, block = 2, 128, 7
    tables = torch.tensor([[4, 2, -1], [0, 9, 3], [1, 5, 8], [6, 7, -1]])
    offsets = torch.tensor([9, 14, 21, 14])  # inside, last page, past the table, on padding
    key, value = (torch.randn(4, heads, dim, generator=gen).bfloat16() for _ in range(2))
    kc, vc = caches(9, heads, block, dim)  # page 9 does not exist
    before = kc.clone()
    write_kv_cache_batch_fp4(kc, vc, tables.to(DEV), offsets.to(DEV), key.to(DEV), value.to(DEV), block,
                             validate=False)
    slots = torch.tensor([2 * block + 2, 3 * block, -1, -1])
    assert torch.equal(kc.cpu(), written(before, key, slots, block))
    assert torch.equal(vc.cpu(), written(before, value, slots, block))
    rows = torch.randn(9 * block, heads, dim, generator=gen).bfloat16()
    write_kv_cache_slots_fp4(kc, vc, torch.arange(9 * block, device=DEV), rows.to(DEV), rows.to(DEV), block)
    ids = torch.tensor([8, 0, 11, 3], device=DEV)
    k, v = gather_kv_cache_fp4(kc, vc, ids, 4 * block - 3, block, dim, torch.bfloat16, validate=False)
    want = f4.values(*f4.quantise(rows)).view(9, block, heads, dim)
    want = torch.cat((want[8], want[0], torch.zeros(block, heads, dim), want[3]))[:-3]
    assert torch.equal(k.cpu().double(), want) and torch.equal(v.cpu().double(), want)


def test_empty_calls_write_nothing():
    kc, vc = caches(2, 2, 16, 32)
    before = kc.clone()
    none = torch.empty(0, 2, 32, dtype=torch.float16, device=DEV)
    ids = torch.empty(0, dtype=torch.int64, device=DEV)
    write_kv_cache_slots_fp4(kc, vc, ids, none, none, 16)
    write_kv_cache_batch_fp4(kc, vc, torch.empty(0, 3, dtype=torch.int64, device=DEV), ids, none, none, 16)
    k, v = gather_kv_cache_slots_fp4(kc, vc, ids, 16, 32, torch.bfloat16)
    assert k.shape == v.shape == (0, 2, 32)
    k, v = gather_kv_cache_fp4(kc, vc, ids, 0, 16, 32, torch.bfloat16)
    assert k.shape == v.shape == (0, 2, 32)
    assert torch.equal(kc, before) and torch.equal(vc, before)


def test_pages_past_four_gigabytes():
    """Byte offsets beyond 32 bits, written and read (and beyond 2^31 slots' worth of dims)."""
    heads, dim, block = 8, 128, 256
    pages = 33000
    kc, vc = (torch.empty(pages, heads, fp4_record_bytes(block, dim), dtype=torch.uint8, device=DEV) for _ in range(2))
    assert kc.numel() > 1 << 32
    gen = torch.Generator().manual_seed(6)
    key, value = (torch.randn(5, heads, dim, generator=gen).half().to(DEV) for _ in range(2))
    slots = torch.tensor([0, 31000 * block + 7, pages * block - 1, 15500 * block, 30841 * block + 255], device=DEV)
    write_kv_cache_slots_fp4(kc, vc, slots, key, value, block)
    k, v = gather_kv_cache_slots_fp4(kc, vc, slots, block, dim, torch.float16)
    assert torch.equal(k.cpu().double(), f4.values(*f4.quantise(key.cpu())))
    assert torch.equal(v.cpu().double(), f4.values(*f4.quantise(value.cpu())))
