"""The native call path of the packed cache's and the page operators' entry
points against the Python path: the same bits for every form it takes, and
None for what it leaves to the Python code."""

import pytest
import torch

import fp4_cases as f4
from mini_engine_hip.kernels import fp4, pages
from mini_engine_hip.kernels import hip_extension as ext

DEV = "cuda"


def arguments(device, dtype=torch.bfloat16, batch=3, heads=4, kv=2, dim=64, block=16):
    gen = torch.Generator().manual_seed(7)
    lens = [1 + 40 * i for i in range(batch)]
    tables, count = f4.tables_of(gen, lens, block)
    kc, vc = f4.random_caches(gen, count, kv, block, dim, dtype)
    q = torch.randn(batch, heads, dim, generator=gen).to(dtype)
    return [t.to(device) for t in (q, kc, vc, tables, torch.tensor(lens))] + [block]


class Subclass(torch.Tensor):
    pass


def test_declines_what_is_not_plain():
    native = ext.native_calls()
    args = arguments("cpu")
    q, kc, vc, tables, lens, block = args
    for name, call in (("fp4_decode", (*args, 0)), ("fp4_prefill", (q, kc, vc, lens, lens, tables, lens, block, 0)),
                       ("fp4_write_slots", (kc, vc, lens, q[:, :2], q[:, :2], block)),
                       ("fp4_write_batch", (kc, vc, tables, lens, q[:, :2], q[:, :2], block)),
                       ("fp4_gather_slots", (kc, vc, lens, block, 64, torch.float16)),
                       ("move_pages", (kc, lens, lens, None, 0)), ("move_pages", (kc, lens, lens, tables, 0))):
        function = getattr(native, name)
        assert function(*call) is None
        assert function() is None
        assert function(call[0].as_subclass(Subclass), *call[1:]) is None
        assert function(None, *call[1:]) is None
        assert function(*call[:-1], "x") is None


@pytest.fixture
def python_path(monkeypatch):
    """A way to make one call on the Python code alone."""
    def run(function, *args, **kw):
        ext.load_hip_extension()
        with monkeypatch.context() as patch:
            patch.setattr(ext, "native", ext.NoNativeCalls())
            return function(*args, **kw)
    return run


@pytest.fixture
def counted(monkeypatch):
    """The native functions, counting the calls that they took."""
    module = ext.native_calls()
    taken = []

    class Counting:
        def __getattr__(self, name):
            def call(*args):
                result = getattr(module, name)(*args)
                if result is not None:
                    taken.append(name)
                return result
            return call

    monkeypatch.setattr(ext, "native", Counting())
    return taken


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_same_bits_as_the_python_path(counted, python_path, dtype):
    q, kc, vc, tables, lens, block = arguments(DEV, dtype)
    want = python_path(fp4.paged_attention_fp4, q, kc, vc, tables, lens, block, validate=False)
    assert torch.equal(fp4.paged_attention_fp4(q, kc, vc, tables, lens, block, validate=False), want)
    cu = torch.arange(4, device=DEV)
    prefill = (q, kc, vc, cu, lens - 1, tables, lens, block)
    want = python_path(fp4.paged_prefill_attention_fp4, *prefill, validate=False)
    assert torch.equal(fp4.paged_prefill_attention_fp4(*prefill, validate=False), want)
    fused = torch.randn(3, 2 * 2 * 64 + 8, dtype=dtype, device=DEV)
    key, value = fused[:, :128].unflatten(1, (2, 64)), fused[:, 128:256].unflatten(1, (2, 64))
    slots = torch.tensor([7, 50, 3], device=DEV)
    copies = [[c.clone() for c in (kc, vc)] for _ in range(4)]
    fp4.write_kv_cache_slots_fp4(*copies[0], slots, key, value, block, validate=False)
    python_path(fp4.write_kv_cache_slots_fp4, *copies[1], slots, key, value, block, validate=False)
    fp4.write_kv_cache_batch_fp4(*copies[2], tables, lens - 1, key, value, block, validate=False)
    python_path(fp4.write_kv_cache_batch_fp4, *copies[3], tables, lens - 1, key, value, block, validate=False)
    assert all(torch.equal(a, b) for i in (0, 2) for a, b in zip(copies[i], copies[i + 1]))
    assert not torch.equal(copies[0][0], kc) and not torch.equal(copies[2][0], kc)
    got = fp4.gather_kv_cache_slots_fp4(*copies[0], slots, block, 64, dtype, validate=False)
    want = python_path(fp4.gather_kv_cache_slots_fp4, *copies[0], slots, block, 64, dtype, validate=False)
    assert all(torch.equal(a, b) and a.shape == (3, 2, 64) and a.dtype == dtype for a, b in zip(got, want))
    src, dst, numbers = torch.tensor([2, 4], device=DEV), torch.tensor([0, 1], device=DEV), tables.clone()
    planes = [torch.stack((kc, vc)) for _ in range(2)]
    pages.copy_kv_pages(planes[0], src, dst, page_dim=1, validate=False)
    python_path(pages.copy_kv_pages, planes[1], src, dst, page_dim=1, validate=False)
    assert torch.equal(*planes)
    pages.compact_kv_pages(planes[0], src + 1, dst, numbers, page_dim=1, validate=False)
    python_path(pages.compact_kv_pages, planes[1], src + 1, dst, tables, page_dim=1, validate=False)
    assert torch.equal(*planes) and torch.equal(numbers, tables)
    assert counted == ["fp4_decode", "fp4_prefill", "fp4_write_slots", "fp4_write_batch", "fp4_gather_slots",
                       "move_pages", "move_pages"]


@pytest.mark.gpu
def test_declines_on_the_gpu_what_the_python_code_prepares_or_refuses(counted):
    q, kc, vc, tables, lens, block = arguments(DEV)
    want = fp4.paged_attention_fp4(q, kc, vc, tables, lens, block)  # validating: not asked
    strided = torch.stack((q, q), -1)[..., 0]
    assert torch.equal(fp4.paged_attention_fp4(strided, kc, vc, tables, lens, block, validate=False), want)
    assert torch.equal(fp4.paged_attention_fp4(q, kc, vc, tables, lens, block, validate=False,
                                               out=torch.empty_like(q)), want)
    for bad in ((q, kc, vc, tables, lens, 8), (q, kc, vc[1:], tables, lens, block), (q[:, :3], kc, vc, tables, lens, block),
                (q, kc, vc, tables.int(), lens, block), (q, kc, vc, tables, lens[1:], block)):
        with pytest.raises(ValueError):
            fp4.paged_attention_fp4(*bad, validate=False)
    with pytest.raises(ValueError):
        pages.copy_kv_pages(kc, lens, lens[1:], validate=False)
    with pytest.raises(ValueError):
        pages.copy_kv_pages(kc.transpose(0, 1), lens, lens, validate=False)
    with pytest.raises(ValueError):
        fp4.write_kv_cache_slots_fp4(kc, vc, lens, q, q, block, validate=False)
    assert counted == []
