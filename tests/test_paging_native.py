"""The calls of a 4-bit cache's step through the extension module (_dk_native) against their Python
path: the same results where the module takes them, and every other call left to Python."""
import sys
from types import SimpleNamespace

import pytest
import torch

import _dk_native
import attention
import extend
import layout
import paging
from dk_lib import DecodeArgumentError


@pytest.fixture
def python_path(monkeypatch):
    """Runs a function with the module switched off."""
    def run(fn):
        with monkeypatch.context() as m:
            m.setattr(paging, "_NATIVE", False)
            m.setattr(paging, "_native", lambda: False)
            return fn()
    return run


def _tables(i64, dev="cuda"):
    it = torch.int64 if i64 else torch.int32
    table = torch.full((6, 9), -7, dtype=torch.int32, device=dev)
    table[:, :3] = torch.arange(18, dtype=torch.int32, device=dev).view(6, 3)
    rows = torch.tensor([4, 0, 5], dtype=it, device=dev)
    cached = torch.tensor([17, 0, 40], dtype=it, device=dev)
    new = torch.tensor([1, 33, 0], dtype=it, device=dev)
    pages = torch.tensor([30, 31, 32], dtype=torch.int32, device=dev)
    return table, rows, cached, new, pages


@pytest.mark.gpu
@pytest.mark.parametrize("i64", [False, True])
def test_tables_are_the_same(python_path, i64):
    a, b = _tables(i64), _tables(i64)
    got = paging.grow_block_tables(*a, 40, 12)
    want = python_path(lambda: paging.grow_block_tables(*b, 40, 12))
    assert torch.equal(a[0], b[0]) and type(got) is type(want)
    total = int(want.kv_indptr[-1])
    for name, x, y in zip(got._fields, got, want):
        n = total if name == "kv_indices" else y.shape[0]
        assert x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride()
        assert torch.equal(x[:n], y[:n]), name
    # the parts are tensors of their own: a write into one leaves the others
    keep = [t.clone() for t in got]
    got.slots.fill_(5)
    got.slots.add_(1)
    assert all(torch.equal(x, y) for n, x, y in zip(got._fields, got, keep)
               if n not in ("slots", "kv_indices"))
    assert bool((got.slots == 6).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rope,i64", [(False, False), (True, False), (True, True)])
def test_rows_are_the_same(python_path, dtype, rope, i64):
    it = torch.int64 if i64 else torch.int32
    g = torch.Generator().manual_seed(3)
    k, v, q = (torch.randn(5, h, 128, generator=g).to(dtype).cuda() for h in (2, 2, 6))
    slots = torch.tensor([3, 64, -1, 17, 1000], dtype=it, device="cuda")
    pos = torch.tensor([0, 7, 100000, 3, 9], dtype=it, device="cuda")
    freq = torch.rand(64, generator=g).cuda() if rope else None

    def run():
        cache = layout.alloc_kv4_cache(8, 2, 128, device="cuda").fill_(0x33)
        mine = q.clone()
        paging.write_kv4(k, v, cache, slots, q=mine, inv_freq=freq,
                         positions=pos if rope else None, rope_style=int(i64))
        return (cache, mine) + tuple(paging.read_kv4(cache, slots, dtype))
    got, want = run(), python_path(run)
    assert len(got) == len(want)
    for x, y in zip(got, want):
        assert x.dtype == y.dtype and x.shape == y.shape and x.is_contiguous()
        assert torch.equal(x, y)


def _prefill(dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(5)
    cache = layout.alloc_kv4_cache(60, 2, 64, device="cuda")
    k = torch.randn(960, 2, 64, generator=g).to(dtype).cuda()
    paging.write_kv4(k, k.flip(0), cache, torch.arange(960, device="cuda"))
    table = torch.arange(60, dtype=torch.int32, device="cuda").view(1, 60).repeat(3, 1)
    return torch.randn(80, 6, 64, generator=g).to(dtype).cuda(), cache, table


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prefill_is_the_same(python_path, dtype):
    q, cache, table = _prefill(dtype)
    sinks = torch.randn(6, device="cuda")
    for kw in (dict(), dict(scale=0.3), dict(logit_cap=0.0, window=0), dict(logit_cap=9.0, window=50, sinks=sinks),
               dict(out=torch.empty(80, 6, 64, dtype=dtype, device="cuda")),
               dict(out=torch.empty(6, 80, 64, dtype=dtype, device="cuda").transpose(0, 1))):
        for args in (([0, 2], [30, 50], [33, 700]), ((1,), (3,), (960,)), ([], [], [])):
            got = extend.extend_attention_kv4(q, cache, table, *args, **kw)
            assert got is kw["out"] if "out" in kw else got.is_contiguous()
            mine = got.clone()
            want = python_path(lambda: extend.extend_attention_kv4(q, cache, table, *args, **kw))
            n = sum(args[1])
            assert torch.equal(mine[:n], want[:n]), (kw, args)


@pytest.mark.gpu
def test_the_module_takes_plain_prefill_calls():
    q, cache, table = _prefill()
    call = (q, cache, table, [0, 2], [30, 50], [33, 700], None, None, None, None, None)
    native = paging._native()
    assert isinstance(native.extend_attention_kv4(*call), torch.Tensor)
    assert native.extend_attention_kv4(*call[:4], [30, 51], *call[5:]) not in (0, None)      # more than q has
    for at, bad in ((0, q.float()), (0, q[..., :32]), (0, q[:, :5]), (1, cache.cpu()), (2, table.long()),
                    (3, [0]), (3, [0, -1]), (3, torch.tensor([0, 2])), (4, [30, 50.0]), (5, [33, 2 ** 40]),
                    (6, torch.empty_like(q).float()), (7, 1), (7, -1.0), (8, -2.0), (9, -3), (9, 2.0),
                    (10, torch.zeros(5, device="cuda"))):
        assert native.extend_attention_kv4(*call[:at], bad, *call[at + 1:]) is None, (at, bad)
    with pytest.raises(DecodeArgumentError):
        extend.extend_attention_kv4(q, cache, table, [0, 2], [30, 51], [33, 700])
    got = extend.extend_attention_kv4(q, cache, table, torch.tensor([0, 2]), [30, 50], [33, 700])
    assert torch.equal(got[:80], native.extend_attention_kv4(*call)[:80])


@pytest.mark.gpu
def test_the_module_takes_the_plain_calls():
    native = paging._native()
    assert native is _dk_native
    table, rows, cached, new, pages = _tables(False)
    assert type(native.grow_block_tables(table, rows, cached, new, pages, 34, 8)) is tuple
    cache = layout.alloc_kv4_cache(4, 1, 64, device="cuda")
    k = torch.randn(3, 1, 64, dtype=torch.float16, device="cuda")
    slots = torch.arange(3, device="cuda")
    write = (k, k.clone(), cache, slots, None, None, None, 0)
    assert native.write_kv4(*write) == 0
    assert type(native.read_kv4(cache, slots, 0)) is tuple
    # not plain: left to Python, which runs or refuses them
    assert native.grow_block_tables(table, rows[:0], cached[:0], new[:0], pages, 34, 8) is None
    assert native.grow_block_tables(table, rows, cached, new, pages, 34.0, 8) is None
    assert native.grow_block_tables(table, rows, cached, new, pages.cpu(), 34, 8) is None
    assert native.grow_block_tables(table.t(), rows, cached, new, pages, 34, 8) is None
    assert native.read_kv4(cache, slots[::2], 0) is None
    assert native.read_kv4(cache, slots.cpu(), 0) is None
    for at, bad in ((0, k.float()), (1, k.cpu()), (2, cache[..., :-1]), (3, slots[:2]), (4, k[:2]),
                    (5, torch.ones(32, device="cuda")), (6, slots.float()), (7, 2), (7, True)):
        assert native.write_kv4(*write[:at], bad, *write[at + 1:]) is None, at
    sub = k.as_subclass(type("Sub", (torch.Tensor,), {}))
    assert native.write_kv4(sub, sub, *write[2:]) is None


@pytest.mark.gpu
def test_the_c_abi_refuses_through_the_module():
    cache = layout.alloc_kv4_cache(4, 1, 64, device="cuda")
    k = torch.randn(3 * 68 + 8, dtype=torch.float16, device="cuda").as_strided((3, 1, 64), (68, 68, 1))
    slots = torch.arange(3, device="cuda")
    assert paging._native().write_kv4(k, k, cache, slots, None, None, None, 0) not in (0, None)
    with pytest.raises(DecodeArgumentError, match="multiples of 8"):
        paging.write_kv4(k, k, cache, slots)


def test_left_to_python_without_a_gpu():
    native = paging._native()
    if native is False:
        pytest.skip("the extension does not fit this interpreter")
    cache = layout.alloc_kv4_cache(4, 1, 64, device="cpu")
    k = torch.zeros(3, 1, 64, dtype=torch.float16)
    slots = torch.arange(3)
    assert native.grow_block_tables(*_tables(False, "cpu"), 34, 8) is None
    assert native.write_kv4(k, k, cache, slots, None, None, None, 0) is None
    assert native.read_kv4(cache, slots, 0) is None
    assert native.grow_block_tables(*(None,) * 7) is None
    assert native.write_kv4(*(None,) * 8) is None and native.read_kv4(*(None,) * 3) is None
    assert native.extend_attention_kv4(*(None,) * 11) is None
    for fn in (native.grow_block_tables, native.write_kv4, native.read_kv4, native.extend_attention_kv4):
        with pytest.raises(TypeError):
            fn(k)


def test_an_extension_without_these_calls_leaves_them_to_python(monkeypatch):
    old = SimpleNamespace(BUILT_FOR=_dk_native.BUILT_FOR, decode=lambda *a: None)
    monkeypatch.setitem(sys.modules, "_dk_native", old)
    monkeypatch.setattr(attention, "_NATIVE", old.decode)
    monkeypatch.setattr(attention, "_bind_native", lambda: old.decode)
    monkeypatch.setattr(paging, "_NATIVE", None)
    assert paging._native() is False
    with pytest.raises(DecodeArgumentError):
        paging.read_kv4(layout.alloc_kv4_cache(4, 1, 64, device="cpu"), torch.arange(2))
