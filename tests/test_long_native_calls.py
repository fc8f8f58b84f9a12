"""The native call path of the long-context operators against the Python path:
the same bits for every form it takes, and None for what it leaves to the
Python code."""

import pytest
import torch

import long_cases as lc
from mini_engine_hip.kernels import evict, shared, weights
from mini_engine_hip.kernels import hip_extension as ext
from test_fp4_native_calls import Subclass, counted, python_path  # noqa: F401  (fixtures)

DEV = "cuda"


def arguments(device, dtype=torch.bfloat16, lens=(41, 300, 17, 90), heads=4, kv=2, dim=64, block=16):
    gen = torch.Generator().manual_seed(7)
    tables, pages = lc.shared_tables(gen, list(lens), block)
    key, value = lc.caches(gen, pages, block, kv, dim, dtype, tables, list(lens))
    q = torch.randn(len(lens), heads, dim, generator=gen).to(dtype)
    account = torch.rand(len(lens), kv, tables.shape[1] * block, generator=gen)
    return [t.to(device) for t in (q, key, value, tables, torch.tensor(lens))] + [block, account.to(device)]


def test_declines_what_is_not_plain():
    native = ext.native_calls()
    q, key, value, tables, lens, block, account = arguments("cpu")
    step = (q, key, value, tables, lens, block)
    for name, call, number in (("shared_prefix", (*step, torch.tensor([0, 4]), torch.tensor([16])), 5),
                               ("decode_weights", (*step, account), 5),
                               ("prefill_weights", (q, key, torch.arange(5), lens - 1, tables, lens, block, account), 6),
                               ("evict", (key, value, account, tables, lens, block, 20, None, 0), 5),
                               ("evict", (key, value, account, tables, lens, block, 20, lens, 0), 5)):
        function = getattr(native, name)
        assert function(*call) is None  # (not on a device)
        assert function() is None
        assert function(call[0].as_subclass(Subclass), *call[1:]) is None
        assert function(None, *call[1:]) is None
        assert function(*call[:-1], "x") is None
        for bad in (None, "x", 16.0, 2 ** 70, True):
            assert function(*call[:number], bad, *call[number + 1:]) is None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_same_bits_as_the_python_path(counted, python_path, dtype):  # noqa: F811
    q, key, value, tables, lens, block, account = arguments(DEV, dtype)
    offsets, prefixes = torch.tensor([0, 2, 4], device=DEV), torch.tensor([0, 0], device=DEV)
    call = (q, key, value, tables, lens, block, offsets, prefixes)
    want = python_path(shared.paged_attention_shared_prefix, *call, validate=False)
    assert torch.equal(shared.paged_attention_shared_prefix(*call, validate=False), want)
    accounts = [account.clone() for _ in range(2)]
    want = python_path(weights.paged_attention_weights, *call[:6], accounts[0], validate=False)
    assert torch.equal(weights.paged_attention_weights(*call[:6], accounts[1], validate=False), want)
    assert torch.equal(*accounts) and not torch.equal(accounts[0], account)
    rows = (q, key, torch.arange(5, device=DEV), lens - 1, tables, lens, block)
    accounts = [account.clone() for _ in range(2)]
    python_path(weights.prefill_attention_weights, *rows, accounts[0], validate=False)
    assert weights.prefill_attention_weights(*rows, accounts[1], validate=False) is None
    assert torch.equal(*accounts) and not torch.equal(accounts[0], account)
    for first, layers in ((None, False), (torch.tensor([1, 20, 3, 0], device=DEV), True)):
        caches = [[c.clone()[None] if layers else c.clone() for c in (key, value)] for _ in range(2)]
        kind = dict(first=first, recent=5, validate=False)
        w = account[None] if layers else account
        want = python_path(evict.evict_kv_cache, *caches[0], w, tables, lens, block, 33, **kind)
        got = evict.evict_kv_cache(*caches[1], w, tables, lens, block, 33, **kind)
        assert all(torch.equal(a, b) and a.dtype == b.dtype and a.shape == b.shape for a, b in zip(got, want))
        # (As bits: pages that nobody holds are NaN.)
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(*caches))
        assert not torch.equal(caches[0][0].view(torch.int16).flatten(), key.view(torch.int16).flatten())
    assert counted == ["shared_prefix", "decode_weights", "prefill_weights", "evict", "evict"]


@pytest.mark.gpu
def test_declines_on_the_gpu_what_the_python_code_prepares_or_refuses(counted):  # noqa: F811
    q, key, value, tables, lens, block, account = arguments(DEV)
    offsets, prefixes = torch.tensor([0, 4], device=DEV), torch.tensor([0], device=DEV)
    step = (q, key, value, tables, lens, block)
    want = shared.paged_attention_shared_prefix(*step, offsets, prefixes)  # validating: not asked
    out = torch.empty_like(q)
    assert torch.equal(shared.paged_attention_shared_prefix(*step, offsets, prefixes, validate=False, out=out), want)
    odd = torch.empty(q.numel() + 4, dtype=q.dtype, device=DEV)[4:].view(q.shape).copy_(q)  # 8 bytes past a 16-byte boundary
    assert torch.equal(shared.paged_attention_shared_prefix(odd, *step[1:], offsets, prefixes, validate=False), want)
    for bad in (offsets[:1], offsets.int(), torch.arange(8, device=DEV)[::4]):
        with pytest.raises(ValueError):
            shared.paged_attention_shared_prefix(*step, bad, prefixes, validate=False)
    for bad in (account[..., :-16].contiguous(), account.double(), account.transpose(0, 1), account[:1],
                key.view(torch.float32).flatten()[:account.numel()].view(account.shape)):
        with pytest.raises((ValueError, RuntimeError)):
            weights.paged_attention_weights(*step, bad, validate=False)
        with pytest.raises(ValueError):
            weights.prefill_attention_weights(q, key, torch.arange(5, device=DEV), lens - 1, tables, lens, block, bad,
                                              validate=False)
        with pytest.raises(ValueError):
            evict.evict_kv_cache(key, value, bad, tables, lens, block, 33, validate=False)
    for change in ((key, key, 33), (key, value, 0), (key, value, True), (key, value[1:], 33)):
        with pytest.raises(ValueError):
            evict.evict_kv_cache(*change[:2], account, tables, lens, block, change[2], validate=False)
    assert counted == []
