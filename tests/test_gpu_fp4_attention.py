"""Decode and prefill attention over packed 4-bit pages, on the GPU, against
float64 with bounds that count the roundings (fp4_cases.attention)."""

import pytest
import torch

import fp4_cases as f4
from mini_engine_hip.kernels import hip_extension as ext
from mini_engine_hip.kernels.fp4 import (fp4_prefill_workspace_bytes, fp4_workspace_bytes, paged_attention_fp4,
                                         paged_prefill_attention_fp4)

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def decode_case(lens, dtype, *, heads=16, kv=8, dim=128, block=16, seed=0, pad=0):
    gen = torch.Generator().manual_seed(seed + 31 * dim + block)
    tables, pages = f4.tables_of(gen, lens, block, pad=pad)
    kc, vc = f4.random_caches(gen, pages, kv, block, dim, dtype)
    query = torch.randn(len(lens), heads, dim, generator=gen).to(dtype)
    return [query, kc, vc, tables, torch.tensor(lens)], block


def run_decode(args, block, **kw):
    return paged_attention_fp4(*[a.to(DEV) for a in args], block, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("block", [16, 256, 7])
def test_decode_head_dims(dtype, dim, block):
    args, block = decode_case((1, 17, 257, 521), dtype, dim=dim, block=block, heads=6, kv=2)
    f4.assert_within(run_decode(args, block), *f4.decode_oracle(*args, block))


@pytest.mark.parametrize("heads,kv", [(8, 8), (14, 2), (16, 1), (17, 1), (40, 2), (33, 1), (24, 3)])
@pytest.mark.parametrize("partition", [0, 64])
def test_decode_groups(heads, kv, partition):
    """Groups that fill a matrix tile, leave columns of it idle, and take several."""
    args, block = decode_case((300, 1, 95), torch.bfloat16, heads=heads, kv=kv, dim=64, seed=heads)
    f4.assert_within(run_decode(args, block, partition_tokens=partition), *f4.decode_oracle(*args, block))


@pytest.mark.parametrize("block,lens", [(1, (3, 70)), (16, (16, 32, 33)), (24, (70, 24)), (256, (255, 256, 257)),
                                        (5000, (4999,)), (16, (31, 63, 64, 65, 511, 512, 513))])
def test_decode_block_and_tile_boundaries(block, lens):
    args, block = decode_case(lens, torch.float16, block=block, heads=4, kv=2)
    want = f4.decode_oracle(*args, block)
    for partition in (0, 32, 96, 4096):
        f4.assert_within(run_decode(args, block, partition_tokens=partition), *want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("partition", [0, 32])
def test_decode_empty_sequences_and_absent_pages(dtype, partition):
    """Lengths that give no keys, pages that do not exist (a whole sequence of them too), trusted metadata."""
    args, block = decode_case((40, 100, 130, 64, 9, 50), dtype, heads=8, kv=2, pad=2)
    tables, lens = args[3], args[4]
    lens[1], lens[4], lens[3] = 0, -7, (tables.shape[1] * block) + 1
    tables[2, 3], tables[2, 5], tables[2, 8] = -1, 1 << 40, args[1].shape[0]
    tables[5] = -1
    want = f4.decode_oracle(*args, block)
    got = run_decode(args, block, validate=False, partition_tokens=partition)
    f4.assert_within(got, *want)
    assert not got[[1, 3, 4, 5]].any()


def test_decode_ignores_what_is_behind_the_length():
    """Bytes behind a sequence's last token, whatever they are, change nothing; so does the padding."""
    args, block = decode_case((33, 5), torch.bfloat16, heads=8, kv=2, dim=96, block=7)
    base = run_decode(args, block)
    for fill in (0xFF, 0xFE, 0x00):
        dirty = [args[0], *(torch.full_like(c, fill) for c in args[1:3]), *args[3:]]
        for cache, clean in zip(dirty[1:3], args[1:3]):
            code, byte = f4.split(clean, block, 96)
            dcode, dbyte = f4.split(cache, block, 96)
            for b, n in enumerate(args[4].tolist()):
                for t in range(n):
                    page = args[3][b, t // block]
                    dcode[page, :, t % block], dbyte[page, :, t % block] = code[page, :, t % block], byte[page, :, t % block]
            cache.copy_(f4.join(dcode, dbyte))
            cache[..., block * (96 // 2 + 96 // 32):] = fill
        assert torch.equal(run_decode(dirty, block), base)


@pytest.mark.parametrize("dtype", TYPES)
def test_decode_extreme_values(dtype):
    """Scores in the hundreds, rising with the position, tiny and large values: the running reference moves."""
    gen = torch.Generator().manual_seed(8)
    n, dim, block = 700, 128, 16
    tables, pages = f4.tables_of(gen, (n,), block)
    rows = torch.randn(pages, 2, block, dim, generator=gen)
    for at in range(n):
        rows[tables[0, at // block], :, at % block] += at / 100
    kc = f4.packed((rows * 3).to(dtype))
    for size in (2.0 ** -20, 1.0, 40000.0):
        vc = f4.packed((torch.randn(pages, 2, block, dim, generator=gen) * size).clamp(-60000, 60000).to(dtype))
        query = torch.cat((torch.ones(1, 2, dim), -torch.ones(1, 2, dim)), 1).to(dtype) * 2
        args = [query, kc, vc, tables, torch.tensor([n])]
        want = f4.decode_oracle(*args, block)
        for partition in (0, 64):
            f4.assert_within(run_decode(args, block, partition_tokens=partition), *want)


def test_decode_nan_blocks_reach_the_sequences_that_hold_them():
    args, block = decode_case((70, 70), torch.float16, heads=4, kv=2, dim=64)
    code, byte = f4.split(args[2], block, 64)
    byte[args[3][0, 2], 1, 5] = 255  # sequence 0, kv head 1, token 37
    args[2] = f4.join(code, byte)
    got = run_decode(args, block)
    assert got[0, 2:].isnan().all() and not got[0, :2].isnan().any() and not got[1].isnan().any()
    code, byte = f4.split(args[1], block, 64)
    byte[args[3][1, 0], 0, 0, 1] = 255
    args[1] = f4.join(code, byte)
    got = run_decode(args, block)
    assert got[1, :2].isnan().all() and not got[1, 2:].isnan().any()


def test_decode_keeps_a_nan_value_block_to_its_dims():
    args, block = decode_case((70, 70), torch.float16, heads=4, kv=2, dim=64)
    clean = run_decode(args, block)
    code, byte = f4.split(args[2], block, 64)
    byte[args[3][0, 2], 1, 5, 1] = 255  # sequence 0, kv head 1, token 37, dims 32 .. 63
    args[2] = f4.join(code, byte)
    got = run_decode(args, block)
    assert got[0, 2:, 32:].isnan().all()
    got[0, 2:, 32:] = clean[0, 2:, 32:]
    assert torch.equal(got, clean)


def test_decode_long_sequence_and_many_partitions():
    args, block = decode_case((70001,), torch.bfloat16, heads=4, kv=1, block=256)
    want = f4.decode_oracle(*args, block)
    for partition in (0, 32, 1000):
        f4.assert_within(run_decode(args, block, partition_tokens=partition), *want)


def test_decode_is_repeatable_and_takes_buffers():
    args, block = decode_case((900, 31, 400), torch.bfloat16)
    dev = [a.to(DEV) for a in args]
    base = paged_attention_fp4(*dev, block)
    need = fp4_workspace_bytes(3, 16, 8, 128, block, args[3].shape[1])
    out, workspace = torch.empty_like(dev[0]), torch.full((need + 64,), 255, dtype=torch.uint8, device=DEV)
    for _ in range(3):
        assert paged_attention_fp4(*dev, block, out=out, workspace=workspace) is out
        assert torch.equal(out, base)
    strided = torch.empty(3, 16, 256, dtype=torch.bfloat16, device=DEV)[..., ::2]
    strided.copy_(dev[0])
    shifted = torch.empty(3 * 16 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(3, 16, 128)
    shifted.copy_(dev[0])
    assert torch.equal(paged_attention_fp4(strided, *dev[1:], block), base)
    assert torch.equal(paged_attention_fp4(shifted, *dev[1:], block), base)


def test_decode_pages_past_four_gigabytes():
    gen = torch.Generator().manual_seed(9)
    block, dim, kv, pages = 256, 128, 8, 33000
    kc, vc = (torch.empty(pages, kv, f4.record_bytes(block, dim), dtype=torch.uint8, device=DEV) for _ in range(2))
    small = f4.random_caches(gen, 3, kv, block, dim, torch.bfloat16)
    where = torch.tensor([[32999, 17, 31111]])
    for cache, source in zip((kc, vc), small):
        cache[where[0].to(DEV)] = source.to(DEV)
    query = torch.randn(1, 8, dim, generator=gen).bfloat16()
    lens = torch.tensor([700])
    got = paged_attention_fp4(query.to(DEV), kc, vc, where.to(DEV), lens.to(DEV), block)
    f4.assert_within(got, *f4.decode_oracle(query, *small, torch.tensor([[0, 1, 2]]), lens, block))
    got = paged_prefill_attention_fp4(query.to(DEV), kc, vc, torch.tensor([0, 1], device=DEV),
                                      torch.tensor([699], device=DEV), where.to(DEV), lens.to(DEV), block)
    f4.assert_within(got, *f4.decode_oracle(query, *small, torch.tensor([[0, 1, 2]]), lens, block))


# ---------------------------------------------------------------------------
# Prefill
# ---------------------------------------------------------------------------
def prefill_case(new, prior, dtype, *, heads=4, kv=2, dim=128, block=16, seed=0, pad=0):
    gen = torch.Generator().manual_seed(seed + 31 * dim + block)
    lens = [n + p for n, p in zip(new, prior)]
    tables, pages = f4.tables_of(gen, lens, block, pad=pad)
    kc, vc = f4.random_caches(gen, pages, kv, block, dim, dtype)
    query = torch.randn(sum(new), heads, dim, generator=gen).to(dtype)
    cu = torch.tensor([0, *new]).cumsum(0)
    return [query, kc, vc, cu, torch.tensor(prior), tables, torch.tensor(lens)], block


def run_prefill(args, block, **kw):
    return paged_prefill_attention_fp4(*[a.to(DEV) for a in args], block, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("block", [16, 256, 7])
def test_prefill_head_dims(dtype, dim, block):
    args, block = prefill_case((33, 1, 70), (0, 130, 61), dtype, dim=dim, block=block)
    f4.assert_within(run_prefill(args, block), *f4.prefill_oracle(*args, block))


@pytest.mark.parametrize("heads,kv", [(8, 8), (14, 2), (16, 1), (7, 1), (40, 2), (130, 1)])
@pytest.mark.parametrize("chunk", [0, 64])
def test_prefill_groups(heads, kv, chunk):
    """Groups that divide the row tiles, do not, and pass them."""
    args, block = prefill_case((50, 3), (20, 100), torch.bfloat16, heads=heads, kv=kv, dim=32, seed=heads)
    f4.assert_within(run_prefill(args, block, chunk_tokens=chunk), *f4.prefill_oracle(*args, block))


@pytest.mark.parametrize("new,prior", [((1,), (0,)), ((64,), (0,)), ((65, 64, 63), (0, 1, 63)), ((128, 129), (128, 0)),
                                       ((1, 1, 1, 1), (0, 62, 63, 64)), ((0, 5, 0), (0, 3, 0)), ((200,), (333,))])
@pytest.mark.parametrize("chunk", [0, 64, 100])
def test_prefill_row_and_key_boundaries(new, prior, chunk):
    args, block = prefill_case(new, prior, torch.float16, block=16)
    f4.assert_within(run_prefill(args, block, chunk_tokens=chunk), *f4.prefill_oracle(*args, block))


@pytest.mark.parametrize("chunk", [0, 64])
def test_prefill_rows_without_keys(chunk):
    """Absent pages, lengths that do not fit the rows, rows of no sequence: zeros, with trusted metadata."""
    args, block = prefill_case((20, 30, 40, 10, 25), (50, 0, 7, 3, 0), torch.bfloat16, dim=64, pad=1)
    query, _, _, cu, starts, tables, lens = args
    lens[0] = 60            # ten rows past it
    starts[2] = -1
    lens[3] = tables.shape[1] * block + 1
    tables[4] = -1          # no page at all
    tables[1, 0] = 1 << 33  # the first sixteen keys: rows 0..15 see none
    args[0] = torch.cat((query, query[:9]))  # rows behind the last sequence
    want = f4.prefill_oracle(*args, block)
    got = run_prefill(args, block, validate=False, chunk_tokens=chunk)
    f4.assert_within(got, *want)
    assert not got[10:36].any() and not got[50:].any()
    args[3] = cu.clone()
    args[3][0] = 4          # rows before the first sequence
    got = run_prefill(args, block, validate=False, chunk_tokens=chunk)
    assert not got[:4].any()


def test_prefill_offsets_out_of_order_stay_in_bounds():
    args, block = prefill_case((31, 20, 20), (9, 3, 10), torch.bfloat16)
    for cu in ([0, 50, 30, 71], [0, 50, 1 << 40, 71], [-5, 20, 60, 1 << 33], [71, 71, 0, 3]):
        args[3] = torch.tensor(cu)
        for chunk in (0, 64):
            out = run_prefill(args, block, validate=False, chunk_tokens=chunk)
            torch.cuda.synchronize()
            assert out.shape == args[0].shape


@pytest.mark.parametrize("chunk", [0, 64])
def test_prefill_offsets_that_fall_name_too_many_rows(chunk):
    """More row blocks than work-groups: what rows get is open, but every access stays in bounds."""
    args, block = prefill_case((300,) + (0,) * 8, (9,) * 9, torch.bfloat16)
    args[3] = torch.tensor([0, 300] * 5)
    args[6] = torch.full((9,), int(args[6].max()))
    out = run_prefill(args, block, validate=False, chunk_tokens=chunk)
    torch.cuda.synchronize()
    assert out.shape == args[0].shape


@pytest.mark.parametrize("chunk", [0, 64])
@pytest.mark.parametrize("new,prior,cu", [((31, 20, 20), (9, 3, 10), (0, 50, 30, 71)),
                                          ((31, 20, 20), (9, 3, 10), (0, 50, 1 << 40, 71)),
                                          ((31, 20, 20), (9, 3, 10), (-5, 20, 60, 1 << 33)),
                                          ((31, 20, 20), (9, 3, 10), (71, 71, 0, 3)),
                                          ((300,) + (0,) * 8, (9,) * 9, (0, 300) * 5)])
def test_prefill_writes_nothing_beside_its_buffers_whatever_the_offsets(new, prior, cu, chunk):
    """Offsets out of order: the bytes around the output and the workspace stay, and rows with one owner
    are right where there are no more row blocks than work-groups (all but the last case)."""
    args, block = prefill_case(new, prior, torch.bfloat16)
    args[3] = torch.tensor(cu)
    query, kc, vc, offsets, starts, tables, lens = [a.to(DEV) for a in args]
    total, seqs = query.shape[0], len(new)
    lib = ext.load_hip_extension()
    need = lib.fp4_prefill_workspace_size(seqs, total, 4, 2, 128, block, tables.shape[1], chunk)
    out = torch.full((2048 + total * 512 + 2048,), 77, dtype=torch.int16, device=DEV)
    workspace = torch.full((4096 + need + 4096,), 77, dtype=torch.uint8, device=DEV)
    lib.call("mvme_fp4_paged_prefill_attention", out[2048:].data_ptr(), query.data_ptr(), kc.data_ptr(), vc.data_ptr(),
             offsets.data_ptr(), starts.data_ptr(), tables.data_ptr(), lens.data_ptr(), seqs, total, 4, 2, 128,
             kc.shape[0], block, tables.shape[1], chunk, ext.dtype_code(query.dtype), workspace[4096:].data_ptr(), need,
             ext.current_stream(query.device))
    torch.cuda.synchronize()
    assert (out[:2048] == 77).all() and (out[2048 + total * 512:] == 77).all()
    assert (workspace[:4096] == 77).all() and (workspace[4096 + need:] == 77).all()
    clamped = [min(max(c, 0), total) for c in cu]
    owners = torch.zeros(total, dtype=torch.int64)
    for low, high in zip(clamped, clamped[1:]):
        owners[low:max(low, high)] += 1
    owners[:clamped[0]] += 1  # rows before the first and behind the last offset are cleared
    owners[max(clamped[0], clamped[-1]):] += 1
    if seqs == 3:
        args[3] = torch.tensor(clamped)
        want, bound = f4.prefill_oracle(*args, block)
        got = out[2048:2048 + total * 512].view(torch.bfloat16).view(total, 4, 128).cpu()
        f4.assert_within(got[owners == 1], want[owners == 1], bound[owners == 1])


@pytest.mark.parametrize("chunk", [0, 64])
@pytest.mark.parametrize("plane", [1, 2])
def test_prefill_nan_behind_the_mask_stays_there(plane, chunk):
    """A NaN block reaches the rows that see its key and no other (in particular not as 0 * NaN)."""
    args, block = prefill_case((100,), (30,), torch.float16, heads=4, kv=2, dim=64)
    clean = run_prefill(args, block, chunk_tokens=chunk)
    code, byte = f4.split(args[plane], block, 64)
    byte[args[5][0, 90 // block], 1, 90 % block, 1] = 255  # kv head 1, key 90: rows from 60 on
    args[plane] = f4.join(code, byte)
    got = run_prefill(args, block, chunk_tokens=chunk)
    assert torch.equal(got[:60], clean[:60]) and torch.equal(got[:, :2], clean[:, :2])
    assert got[60:, 2:].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 128, 256])
def test_a_key_far_above_the_earlier_ones_at_every_place(dtype, dim):
    """One key whose score is hundreds above all before it: 130 sequences, another place in each, for prefill rows
    before, at and behind it, and for decode.

    The bounds of ``attention`` count what is relative to a probability. Here most are below fp16's range: its
    smallest step is 2^-24, so rounding is off by up to 2^-25 there, and the largest probability is held as 2^8 or
    more (the reference of the exponentials stays 8 or more below the largest score). Per key this is 2^-33 of the
    largest and so of their sum: 2^-33 * n * max|v| in the sum over the values, and the same again by way of the
    sum of n probabilities that divides it, since the output is at most max|v|.
    """
    gen = torch.Generator().manual_seed(13)
    block, tokens, count = 16, 192, 130
    tables, pages = f4.tables_of(gen, (tokens,) * count, block)
    rows = torch.randn(pages, 1, block, dim, generator=gen)
    place = torch.arange(count) + 50
    page = tables[torch.arange(count), place // block]
    rows[page, 0, place % block] = 40.0
    kc, vc = f4.packed(rows.to(dtype)), f4.packed(torch.randn(pages, 1, block, dim, generator=gen).to(dtype))
    lens = torch.full((count,), tokens)
    query = torch.rand(count, 1, dim, generator=gen).to(dtype)
    args = [query, kc, vc, tables, lens]
    floor = 2 * 2.0 ** -33 * tokens * f4.cache_values(vc, block, dim).abs().max()
    want, bound = f4.decode_oracle(*args, block)
    f4.assert_within(run_decode(args, block), want, bound + floor)
    lens = place + 3  # rows at place - 1 .. place + 2
    query = torch.rand(4 * count, 1, dim, generator=gen).to(dtype)
    args = [query, kc, vc, torch.arange(count + 1) * 4, lens - 4, tables, lens]
    want, bound = f4.prefill_oracle(*args, block)
    f4.assert_within(run_prefill(args, block), want, bound + floor)


def test_prefill_many_sequences():
    gen = torch.Generator().manual_seed(11)
    new = torch.randint(0, 9, (150,), generator=gen).tolist()
    prior = torch.randint(0, 40, (150,), generator=gen).tolist()
    new[3] = 90
    prior = [p if n else 0 for n, p in zip(new, prior)]
    args, block = prefill_case(new, prior, torch.bfloat16, dim=32, block=5)
    f4.assert_within(run_prefill(args, block), *f4.prefill_oracle(*args, block))


@pytest.mark.parametrize("chunk", [0, 64])
@pytest.mark.parametrize("count", [2, 63, 64, 65, 129])
def test_prefill_sequence_counts(count, chunk):
    """Row blocks are handed out in two ways, up to 64 sequences and above; some have none, some several."""
    new = [(7 * i * i + 3 * i) % 11 * (i % 5 > 0) + 150 * (i % 40 == 1) for i in range(count)]
    prior = [(13 * i) % 170 for i in range(count)]
    args, block = prefill_case(tuple(new), tuple(prior), torch.bfloat16, heads=4, kv=1, dim=32)
    f4.assert_within(run_prefill(args, block, validate=False, chunk_tokens=chunk), *f4.prefill_oracle(*args, block))


def test_prefill_of_single_rows_equals_decode():
    """One new token per sequence is a decode step: both kernels are within their bounds of each other."""
    args, block = decode_case((1, 300, 77), torch.bfloat16)
    query, kc, vc, tables, lens = args
    want, bound = f4.decode_oracle(*args, block)
    got = run_prefill([query, kc, vc, torch.arange(4), lens - 1, tables, lens], block)
    f4.assert_within(got, want, bound)


def test_prefill_takes_a_workspace():
    args, block = prefill_case((40, 60), (900, 500), torch.bfloat16, heads=16, kv=8)
    dev = [a.to(DEV) for a in args]
    base = paged_prefill_attention_fp4(*dev, block)
    need = fp4_prefill_workspace_bytes(2, 100, 16, 8, 128, block, args[5].shape[1])
    assert need > 0
    workspace = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(paged_prefill_attention_fp4(*dev, block, workspace=workspace), base)


# ---------------------------------------------------------------------------
# Streams and graphs
# ---------------------------------------------------------------------------
def test_other_stream_sees_its_own_order():
    args, block = decode_case((500, 40), torch.float16)
    dev = [a.to(DEV) for a in args]
    base = paged_attention_fp4(*dev, block)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = dev[0] * 0
        torch.cuda._sleep(2_000_000)
        late += dev[0]
        got = paged_attention_fp4(late, *dev[1:], block, validate=False)
    side.synchronize()
    assert torch.equal(got, base)


def test_graph_replays_follow_their_inputs():
    """A captured decode step and prefill: new lengths, tables and queries before every replay."""
    args, block = decode_case((800, 800, 800), torch.bfloat16, seed=5)
    dev = [a.to(DEV) for a in args]
    cu = torch.arange(4, device=DEV)
    starts = dev[4] - 1

    def step():
        return (paged_attention_fp4(*dev, block, validate=False),
                paged_prefill_attention_fp4(*dev[:3], cu, starts, *dev[3:], block, validate=False))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    gen = torch.Generator().manual_seed(12)
    for lens in ((1, 800, 33), (0, 5, 640), (799, 256, 257), (32, 31, 1)):
        dev[0].copy_(torch.randn(3, 16, 128, generator=gen).bfloat16())
        dev[3].copy_(dev[3][torch.randperm(3, generator=gen).to(DEV)].clone())
        dev[4].copy_(torch.tensor(lens))
        starts.copy_(dev[4] - 1)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))


# ---------------------------------------------------------------------------
# Rounded probabilities and their sum
# ---------------------------------------------------------------------------
def equal_values_case(n, heads, dim, seed):
    """n keys of which the first is another than the equal rest, every value 4, one kv head."""
    gen = torch.Generator().manual_seed(seed)
    tables, pages = f4.tables_of(gen, (n,), 16)
    keys = torch.zeros(pages, 1, 16, dim) + torch.randn(dim, generator=gen)
    keys[tables[0, 0], 0, 0] = torch.randn(dim, generator=gen)
    kc, vc = f4.packed(keys.half()), f4.packed(torch.full((pages, 1, 16, dim), 4.0).half())
    return torch.randn(1, heads, dim, generator=gen).half(), kc, vc, tables, torch.tensor([n])


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_average_of_equal_values_is_that_value(dim):
    """Whatever a probability is rounded to, the sum that divides counts it as rounded: 200 queries, 32 keys.

    What is left is the error of fp32 sums of 32 terms, 2^-24 * 64 at most, and fp16 has its next value 2^-11 below 4.
    """
    query, kc, vc, tables, lens = equal_values_case(32, 200, dim, dim)
    assert (run_decode([query, kc, vc, tables, lens], 16) == 4).all()
    assert (run_prefill([query, kc, vc, torch.tensor([0, 1]), lens - 1, tables, lens], 16) == 4).all()


def test_average_of_equal_values_with_most_keys_far_below_one():
    """8191 keys at 2^-23 of the first, which fp16 holds as subnormals: they count in both sums, or in neither.

    A lane adds at most 2048 pairs to the sum and 512 products to the values, each off by 2^-24 of it: 2^-12.7 in
    all, and from 2^-12 on the result would round to the value below 4.  Lost on one side alone they would be 2^-10.
    """
    n, dim = 8192, 64
    gen = torch.Generator().manual_seed(1)
    tables, pages = f4.tables_of(gen, (n,), 16)
    keys = torch.zeros(pages, 1, 16, dim)
    keys[tables[0, 0], 0, 0] = 2.0
    kc, vc = f4.packed(keys.half()), f4.packed(torch.full((pages, 1, 16, dim), 4.0).half())
    query, lens = torch.ones(1, 1, dim).half(), torch.tensor([n])
    assert (run_decode([query, kc, vc, tables, lens], 16, partition_tokens=n) == 4).all()
    args = [query, kc, vc, torch.tensor([0, 1]), lens - 1, tables, lens]
    assert (run_prefill(args, 16, chunk_tokens=n) == 4).all()


@pytest.mark.parametrize("start", [70 - (1 << 32), (1 << 32) + 70, -(1 << 63), (1 << 63) - 1, -1])
def test_prefill_starts_that_cannot_be_see_no_keys(start):
    """Nor do their rows take anything from the workspace: 70 alone would be a key of the second chunk."""
    args, block = prefill_case((40, 20), (200, 100), torch.bfloat16)
    args[4][0] = start
    workspace = torch.ones(fp4_prefill_workspace_bytes(2, 60, 4, 2, 128, block, args[5].shape[1], 64) // 4, device=DEV)
    got = run_prefill(args, block, validate=False, chunk_tokens=64, workspace=workspace)
    f4.assert_within(got, *f4.prefill_oracle(*args, block))
    assert not got[:40].any() and got[40:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", [1, -1])
def test_scores_up_to_nine_million(dtype, order):
    """Keys at 1 and 1.5 times the powers of two up to 2^15, rising or falling: the largest score of a row is 8.9e6.

    Where it is 100 or more above the next (fp32 sums are off by 2^-23 * 272 of it, the next is a quarter below),
    no other key counts, and the output is its value.
    """
    gen = torch.Generator().manual_seed(17)
    n, dim, block = 64, 128, 16
    tables, pages = f4.tables_of(gen, (n,), block)
    at = torch.arange(n)
    size = (1.0 + 0.5 * (at % 2)) * torch.exp2(at // 2 - 16.0)
    size = size if order == 1 else size.flip(0)
    rows = torch.zeros(pages, 1, block, dim)
    rows[tables[0, at // block], 0, at % block] = size[:, None].expand(n, dim)
    kc, vc = f4.packed(rows.to(dtype)), f4.packed(torch.randn(pages, 1, block, dim, generator=gen).to(dtype))
    values = f4.cache_values(vc, block, dim)[tables[0, at // block], at % block, 0]
    scores = 16.0 * dim ** 0.5 * size
    assert 8.8e6 < scores.max() < 9e6
    best = torch.tensor([int(scores[:t + 1].argmax()) for t in range(n)])
    clear = torch.tensor([t > 0 and scores[:t + 1].topk(2).values.diff().item() <= -100 for t in range(n)])
    # Rising, the gap at t is 90 * 2^(t // 2 - 16) for odd t and half of it for even ones: 100 or more from t = 35 on.
    assert clear.sum() == (29 if order == 1 else 63)
    query = torch.full((n, 1, dim), 16.0).to(dtype)
    wide = tables.expand(n, -1).contiguous()
    got = run_decode([query, kc, vc, wide, at + 1], block).cpu().double()[:, 0]
    assert torch.equal(got[clear], values[best[clear]])
    for chunk in (0, 64):
        args = [query, kc, vc, torch.tensor([0, n]), torch.tensor([0]), tables, torch.tensor([n])]
        got = run_prefill(args, block, chunk_tokens=chunk).cpu().double()[:, 0]
        assert torch.equal(got[clear], values[best[clear]])
