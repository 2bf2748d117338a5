"""Serving operators without a GPU: schemas, refusals with their messages, FakeTensor shapes, C entries' checks, and the
plain page model against a direct simulation."""

from __future__ import annotations

import ctypes
import os
import random
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from flux_amd import _native, ops
from flux_amd.ops import serving
from oracle import serving as ref
from tests.conftest import ROOT


def _paged(batch=2, heads=6, kv_heads=2, dim=16, pages=5, page_size=4, columns=3, dtype=torch.float32):
    return {"query": torch.zeros(batch, heads, 1, dim, dtype=dtype),
            "key_pages": torch.zeros(pages, kv_heads, page_size, dim, dtype=dtype),
            "value_pages": torch.zeros(pages, kv_heads, page_size, dim, dtype=dtype),
            "page_table": torch.zeros(batch, columns, dtype=torch.int32),
            "lengths": torch.ones(batch, dtype=torch.int64), "scale": 0.25}


def _window(batch=2, heads=6, kv_heads=2, queries=3, keys=5, dim=16, dtype=torch.float32):
    return {"query": torch.zeros(batch, heads, queries, dim, dtype=dtype),
            "key": torch.zeros(batch, kv_heads, keys, dim, dtype=dtype),
            "value": torch.zeros(batch, kv_heads, keys, dim, dtype=dtype), "scale": 0.25, "window": 4}


def _books(slots=3, columns=4, pages=7):
    return {"page_table": torch.full((slots, columns), -1, dtype=torch.int32),
            "lengths": torch.zeros(slots, dtype=torch.int64), "refcounts": torch.zeros(pages, dtype=torch.int32)}


def _pools(pages=7, kv_heads=2, page_size=4, dim=8, layers=None):
    shape = (pages, kv_heads, page_size, dim) if layers is None else (layers, pages, kv_heads, page_size, dim)
    return {"key_pages": torch.zeros(shape), "value_pages": torch.zeros(shape)}


ids = torch.tensor([0, 1])
CALLS = {
    "paged_decode_attention": lambda: _paged(),
    "paged_decode_attention_out": lambda: {**_paged(), "window": 0, "sinks": 0, "slots": None,
                                           "output": torch.zeros(2, 6, 1, 16), "workspace": torch.zeros(1000)},
    "window_attention": lambda: _window(),
    "paged_cache_reserve": lambda: {**_books(), "page_size": 4, "slots": ids},
    "paged_cache_write": lambda: {"key": torch.zeros(2, 2, 3, 8), "value": torch.zeros(2, 2, 3, 8), **_pools(),
                                  "page_table": _books()["page_table"], "slots": ids, "positions": ids},
    "paged_cache_copy": lambda: {**_pools(layers=2), "source": ids, "target": ids + 2},
    "paged_cache_fork": lambda: {**_pools(layers=2), **_books(), "parents": ids[:1], "children": ids[1:]},
    "paged_cache_free": lambda: {**_books(), "slots": ids},
    "paged_cache_compact": lambda: {**_pools(), "page_table": _books()["page_table"],
                                    "refcounts": _books()["refcounts"]},
    "logits_process": lambda: {"logits": torch.zeros(2, 100), "history": torch.zeros(2, 5, dtype=torch.int64)},
}


def test_every_operator_is_registered_and_exported():
    assert set(CALLS) == set(ops.SERVING_OPERATOR_NAMES) == set(serving.SERVING_SCHEMAS)
    for name in ops.SERVING_OPERATOR_NAMES:
        assert hasattr(torch.ops.flux, name)
    for name in ("paged_decode_attention_native", "paged_decode_attention_native_out", "window_attention_native",
                 "paged_cache_reserve_native", "paged_cache_write_native", "paged_cache_copy_native",
                 "paged_cache_fork_native", "paged_cache_free_native", "paged_cache_compact_native",
                 "logits_process_native"):
        assert name in ops.__all__ and callable(getattr(ops, name))
    assert ops.native_paged_decode_attention_is_available() and ops.native_window_attention_is_available()
    assert ops.native_paged_cache_is_available() and ops.native_logits_process_is_available()


@pytest.mark.parametrize("name", sorted(CALLS))
def test_valid_cpu_tensors_are_refused_for_want_of_a_kernel(name):
    with pytest.raises(RuntimeError, match="no CPU kernel"):
        getattr(torch.ops.flux, name)(**CALLS[name]())


i64, i32, f32 = torch.int64, torch.int32, torch.float32
REFUSED = [
    ("paged_decode_attention", {"query": torch.zeros(2, 6, 16)}, "rank four"),
    ("paged_decode_attention", {"query": torch.zeros(2, 6, 2, 16)}, "query length must be one"),
    ("paged_decode_attention", {"query": torch.zeros(2, 6, 1, 16, dtype=torch.float64)}, "share dtype"),
    ("paged_decode_attention", {"value_pages": torch.zeros(5, 2, 4, 16, dtype=torch.float16)}, "share dtype"),
    ("paged_decode_attention", {"value_pages": torch.zeros(5, 2, 3, 16)}, "page shapes must match"),
    ("paged_decode_attention", {"query": torch.zeros(2, 5, 1, 16)}, "divisible by KV heads"),
    ("paged_decode_attention", {"query": torch.zeros(2, 6, 1, 8)}, "head dimensions must match"),
    ("paged_decode_attention", {**_paged(dim=257)}, "at most 256"),
    ("paged_decode_attention", {"query": torch.zeros(0, 6, 1, 16)}, "non-empty"),
    ("paged_decode_attention", {"page_table": torch.zeros(2, 3, dtype=i64)}, "page_table must be int32"),
    ("paged_decode_attention", {"page_table": torch.zeros(3, 2, dtype=i32).t()}, "rows must be contiguous"),
    ("paged_decode_attention", {"page_table": torch.zeros(2, 1, dtype=i32).expand(2, 5000000)}, "must be contiguous|16777216"),
    ("paged_decode_attention", {"page_table": torch.zeros(3, 3, dtype=i32)}, "one entry per page_table row"),
    ("paged_decode_attention", {"page_table": torch.zeros(3, 3, dtype=i32), "lengths": torch.zeros(3, dtype=i64)},
     "one row per sequence"),
    ("paged_decode_attention", {"lengths": torch.ones(2, dtype=i32)}, "contiguous int64 vector"),
    ("paged_decode_attention", {"lengths": torch.ones(4, dtype=i64)[::2]}, "contiguous int64 vector"),
    ("paged_decode_attention", {"slots": torch.zeros(3, dtype=i64)}, "slots must have one entry"),
    ("paged_decode_attention", {"slots": torch.zeros(2, dtype=i32)}, "slots must be a contiguous int64"),
    ("paged_decode_attention", {"key_pages": torch.zeros(5, 2, 16, 4).transpose(2, 3)}, "unit stride"),
    ("paged_decode_attention", {"window": -1}, "window and sinks"),
    ("paged_decode_attention", {"sinks": -1}, "window and sinks"),
    ("paged_decode_attention", {"scale": float("nan")}, "finite FP32"),
    ("paged_decode_attention", {"query": torch.zeros(2, 6, 1, 16, requires_grad=True)}, "inference-only"),
    ("paged_decode_attention_out", {"output": torch.zeros(2, 6, 1, 15)}, "output must be contiguous"),
    ("paged_decode_attention_out", {"output": torch.zeros(2, 6, 1, 16, dtype=torch.float16)}, "output must be contiguous"),
    ("paged_decode_attention_out", {"workspace": torch.zeros(1000, dtype=torch.float64)}, "workspace must be contiguous"),
    ("window_attention", {"query": torch.zeros(2, 6, 16)}, "rank four"),
    ("window_attention", {"query": torch.zeros(2, 6, 3, 16, dtype=torch.int32)}, "share dtype"),
    ("window_attention", {"value": torch.zeros(2, 2, 4, 16)}, "key and value shapes"),
    ("window_attention", {"query": torch.zeros(2, 6, 0, 16)}, "non-empty"),
    ("window_attention", {"query": torch.zeros(1, 6, 3, 16)}, "batch sizes"),
    ("window_attention", {"query": torch.zeros(2, 7, 3, 16)}, "divisible"),
    ("window_attention", {**_window(dim=264)}, "at most 256"),
    ("window_attention", {"key": torch.zeros(2, 2, 16, 5).transpose(2, 3)}, "unit stride"),
    ("window_attention", {"lengths": torch.zeros(3, dtype=i64)}, "lengths must have one entry"),
    ("window_attention", {"starts": torch.zeros(2, dtype=i32)}, "starts must be a contiguous int64"),
    ("window_attention", {"window": -3}, "window and sinks"),
    ("window_attention", {"scale": float("inf")}, "finite FP32"),
    ("paged_cache_reserve", {"page_size": 0}, "page_size must be positive"),
    ("paged_cache_reserve", {"page_size": 1 << 24}, "at most 16777216"),
    ("paged_cache_reserve", {"page_table": torch.zeros(1, 4, dtype=i32).expand(3, 4)}, "must not overlap"),
    ("paged_cache_reserve", {"lengths": torch.zeros(2, dtype=i64)}, "one entry per page_table row"),
    ("paged_cache_reserve", {"refcounts": torch.zeros(7, dtype=i64)}, "refcounts must be a contiguous int32"),
    ("paged_cache_reserve", {"refcounts": torch.zeros(0, dtype=i32)}, "one entry per page"),
    ("paged_cache_reserve", {"slots": ids.to(i32)}, "slots must be a contiguous int64"),
    ("paged_cache_reserve", {"counts": torch.ones(3, dtype=i64)}, "counts must have one entry"),
    ("paged_cache_write", {**_pools(layers=2)}, r"must be \[pages"),
    ("paged_cache_write", {"key": torch.zeros(2, 2, 4, 8)}, "of one shape"),
    ("paged_cache_write", {"key": torch.zeros(2, 2, 3, 8, dtype=torch.float16)}, "pages' dtype"),
    ("paged_cache_write", {"key": torch.zeros(2, 3, 3, 8), "value": torch.zeros(2, 3, 3, 8)}, "heads and head dimension"),
    ("paged_cache_write", {"key": torch.zeros(2, 2, 8, 3).transpose(2, 3)}, "unit stride"),
    ("paged_cache_write", {"key_pages": torch.zeros(1, 2, 4, 8).expand(7, 2, 4, 8)}, "must not overlap itself"),
    ("paged_cache_write", {"positions": torch.zeros(3, dtype=i64)}, "positions must have one entry"),
    ("paged_cache_write", {"counts": torch.zeros(2, dtype=i32)}, "counts must be a contiguous int64"),
    ("paged_cache_copy", {"target": torch.tensor([1])}, "one length"),
    ("paged_cache_copy", {"source": ids.float()}, "source must be a contiguous int64"),
    ("paged_cache_copy", {"value_pages": torch.zeros(2, 7, 2, 4, 9)}, "page shapes must match"),
    ("paged_cache_fork", {"refcounts": torch.zeros(6, dtype=i32)}, "refcounts must have one entry per page"),
    ("paged_cache_fork", {"children": ids}, "one length"),
    ("paged_cache_free", {"slots": ids[None]}, "slots must be a contiguous int64"),
    ("paged_cache_compact", {"refcounts": torch.zeros(8, dtype=i32)}, "refcounts must have one entry per page"),
    ("logits_process", {"logits": torch.zeros(100)}, r"\[rows, vocab\]"),
    ("logits_process", {"logits": torch.zeros(0, 100)}, "non-empty"),
    ("logits_process", {"logits": torch.zeros(2, 100, dtype=torch.float64)}, "must have dtype"),
    ("logits_process", {"logits": torch.zeros(100, 2).t()}, "logits rows must be contiguous"),
    ("logits_process", {"history": torch.zeros(2, 5, dtype=i32)}, "history must be int64"),
    ("logits_process", {"history_lengths": torch.zeros(3, dtype=i64)}, "history_lengths must have one entry"),
    ("logits_process", {"history": None, "history_lengths": torch.zeros(2, dtype=i64)}, "needs a history"),
    ("logits_process", {"history": None, "presence": torch.zeros(2)}, "presence needs a history"),
    ("logits_process", {"repetition": torch.zeros(3)}, "repetition must have one entry"),
    ("logits_process", {"frequency": torch.zeros(2, dtype=torch.float64)}, "frequency must be a contiguous float32"),
    ("logits_process", {"bias": torch.zeros(3, 100)}, "bias must be float32"),
    ("logits_process", {"allowed": torch.zeros(2, 3, dtype=i32)}, "allowed must be int32"),
    ("logits_process", {"logits": torch.zeros(2, 100, requires_grad=True)}, "inference-only"),
]


@pytest.mark.parametrize("name,change,message", REFUSED, ids=[f"{n}-{m[:20]}-{i}" for i, (n, _, m) in enumerate(REFUSED)])
def test_refusals(name, change, message):
    with pytest.raises(RuntimeError, match=message):
        getattr(torch.ops.flux, name)(**{**CALLS[name](), **change})


def test_out_variant_refuses_aliases():
    args = CALLS["paged_decode_attention_out"]()
    with pytest.raises(RuntimeError, match="must not alias an input"):
        torch.ops.flux.paged_decode_attention_out(**{**args, "output": args["query"]})
    store = torch.zeros(2 * 6 * 16 + 1000)
    with pytest.raises(RuntimeError, match="output and workspace must not alias"):
        torch.ops.flux.paged_decode_attention_out(**{**args, "output": store[:192].view(2, 6, 1, 16),
                                                     "workspace": store[192:]})


def test_write_refuses_a_source_inside_the_pages():
    args = CALLS["paged_cache_write"]()
    args["key"] = args["key_pages"][:2, :, :3]
    with pytest.raises(RuntimeError, match="must not alias key or value"):
        torch.ops.flux.paged_cache_write(**args)


PAGES_CALLS = ("paged_cache_write", "paged_cache_copy", "paged_cache_fork", "paged_cache_compact")


@pytest.mark.parametrize("name", PAGES_CALLS)
def test_pages_that_are_written_lie_apart(name):
    args = CALLS[name]()
    with pytest.raises(RuntimeError, match="must not be the same memory"):
        getattr(torch.ops.flux, name)(**{**args, "value_pages": args["key_pages"]})
    shape = args["key_pages"].shape
    strides = torch.empty(shape).stride()
    for dimension in range(len(shape) - 1):  # a step that ends inside what lies below it
        short = [step - (i == dimension) for i, step in enumerate(strides)]
        if shape[dimension] > 1:
            with pytest.raises(RuntimeError, match="value_pages must not overlap itself"):
                getattr(torch.ops.flux, name)(**{**args, "value_pages": torch.zeros(4000).as_strided(shape, short)})
    padded = {n: torch.zeros(*shape[:-1], shape[-1] + 3)[..., :-3].transpose(-2, -3).contiguous().transpose(-2, -3)
              for n in ("key_pages", "value_pages")}
    with pytest.raises(RuntimeError, match="no CPU kernel"):
        getattr(torch.ops.flux, name)(**{**args, **padded})


def _side_views(shape):
    """(name, key, value, whether they share memory) of one storage, over the layouts that pools come in."""
    *outer, heads, rows, dim = shape
    count = torch.empty(shape).numel()
    page = heads * rows * dim
    flat = torch.zeros(8 * count + 64)
    halves = flat[: 2 * count].view(2, *shape)
    yield "one after the other", halves[0], halves[1], False
    yield "the other after one", halves[1], halves[0], False
    by_page = flat[: 2 * count].view(*outer, 2, heads, rows, dim)
    yield "interleaved by page", by_page[..., 0, :, :, :], by_page[..., 1, :, :, :], False
    by_row = flat[: 2 * count].view(*outer, heads, rows, 2, dim)
    yield "interleaved by row", by_row[..., 1, :], by_row[..., 0, :], False
    turned = flat[: 2 * count].view(*outer, 2, page)
    yield ("interleaved by page, rows before heads", turned[..., 0, :].unflatten(-1, (heads, rows, dim)),
           turned[..., 1, :].unflatten(-1, (rows, heads, dim)).transpose(-2, -3), False)
    padded = flat[: count // dim * (2 * dim + 5)].view(*outer, heads, rows, 2 * dim + 5)
    yield "interleaved in wider rows", padded[..., :dim], padded[..., dim + 3 : 2 * dim + 3], False
    yield "wider rows that meet", padded[..., : dim], padded[..., dim - 1 : 2 * dim - 1], True
    yield "a page on", flat[:count].view(shape), flat[page : page + count].view(shape), True
    yield "an element on", flat[1 : count + 1].view(shape), flat[:count].view(shape), True
    yield "the last element", flat[:count].view(shape), flat[count - 1 : 2 * count - 1].view(shape), True
    yield "the next element", flat[:count].view(shape), flat[count : 2 * count].view(shape), False
    yield "other strides", flat[:count].view(shape), flat[:count].view(*outer, rows, heads, dim).transpose(-2, -3), True
    by_page = flat[: 2 * count].view(*outer, 2, page)
    yield ("interleaved and half a page on", by_page[..., 0, :].unflatten(-1, (heads, rows, dim)),
           flat[page // 2 : 2 * count + page // 2].view(*outer, 2, page)[..., 1, :].unflatten(-1, (heads, rows, dim)), True)


def _shares_memory(key, value):
    def places(t):
        at = torch.zeros(t.shape, dtype=torch.int64)
        for d, step in enumerate(t.stride()):
            at += (torch.arange(t.shape[d]) * step).view([-1 if i == d else 1 for i in range(t.dim())])
        return set((at + t.storage_offset()).flatten().tolist())

    return bool(places(key) & places(value))


@pytest.mark.parametrize("name", PAGES_CALLS)
def test_pools_that_share_memory_are_refused(name):
    """Interleaved pools stay allowed; two views of one storage that meet in an element are not."""
    args = CALLS[name]()
    for what, key, value, shared in _side_views(tuple(args["key_pages"].shape)):
        assert _shares_memory(key, value) == shared, what
        message = f"{name}: key and value pages must not overlap" if shared else "no CPU kernel"
        with pytest.raises(RuntimeError, match=message):
            getattr(torch.ops.flux, name)(**{**args, "key_pages": key, "value_pages": value})


@pytest.mark.parametrize("name,change,message", [r for r in REFUSED if "requires_grad" not in str(r[1])][::4])
def test_fake_tensors_are_refused_alike(name, change, message):
    mode = FakeTensorMode()
    args = {k: mode.from_tensor(v) if isinstance(v, torch.Tensor) else v for k, v in {**CALLS[name](), **change}.items()}
    with mode, pytest.raises(RuntimeError, match=message):
        getattr(torch.ops.flux, name)(**args)


def test_fake_shapes():
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        def fake(values):
            return {k: mode.from_tensor(v) if isinstance(v, torch.Tensor) else v for k, v in values.items()}

        out = torch.ops.flux.paged_decode_attention(**fake(_paged(dtype=torch.bfloat16)))
        assert out.shape == (2, 6, 1, 16) and out.dtype == torch.bfloat16
        assert torch.ops.flux.window_attention(**fake(_window())).shape == (2, 6, 3, 16)
        positions, status = torch.ops.flux.paged_cache_reserve(**fake(CALLS["paged_cache_reserve"]()))
        assert positions.shape == (2,) and positions.dtype == i64 and status.dtype == i32
        assert torch.ops.flux.paged_cache_copy(**fake(CALLS["paged_cache_copy"]())).dtype == i32
        assert torch.ops.flux.paged_cache_fork(**fake(CALLS["paged_cache_fork"]())).shape == (1,)
        assert torch.ops.flux.paged_cache_free(**fake(CALLS["paged_cache_free"]())).shape == (2,)
        page_map, used = torch.ops.flux.paged_cache_compact(**fake(CALLS["paged_cache_compact"]()))
        assert page_map.shape == (7,) and used.shape == ()
        processed, tokens = torch.ops.flux.logits_process(**fake(CALLS["logits_process"]()))
        assert processed.shape == (2, 100) and tokens.shape == (2,) and tokens.dtype == i64


# --------------------------------------------------------------------------- C entries

def _pool_struct(**change):
    values = dict(key=16, value=16, layers=1, pages=4, heads=2, page_size=4, head_dim=8, dtype=0)
    values.update(change)
    pool = _native.PagePool(**values)
    for i, stride in enumerate((256, 64, 32, 8)):
        pool.key_strides[i] = pool.value_strides[i] = stride
    return ctypes.byref(pool)


def _books_struct(**change):
    values = dict(page_table=16, table_stride=4, slots=2, columns=4, lengths=16, refcounts=16, pages=4, page_size=4)
    values.update(change)
    return ctypes.byref(_native.PageBooks(**values))


def test_c_entries_refuse_before_any_launch():
    lib, some = _native.load(), ctypes.c_void_p(16)  # never dereferenced
    bad = _native.FLUX_ERROR_INVALID_VALUE
    four, three = (ctypes.c_int64 * 4)(64, 16, 16, 1), (ctypes.c_int64 * 3)(64, 32, 16)

    def paged(dtype=0, query=some, table=some, workspace=some, size=1 << 20, scale=1.0, batch=2, heads=6, kv=2, dim=16,
              pages=4, page=4, slots=2, columns=4, window=0, sinks=0):
        return lib.flux_paged_decode_attention(dtype, query, some, some, table, some, None, some, workspace, size, scale,
                                               batch, heads, kv, dim, pages, page, slots, columns, columns, window, sinks,
                                               four, three, three, None)

    for change, message in (({"query": None}, "null"), ({"table": None}, "null"), ({"workspace": None}, "null"),
                            ({"dtype": 3}, "dtype"), ({"batch": 0}, "shape"), ({"heads": 5}, "shape"),
                            ({"dim": 257}, "shape"), ({"pages": 0}, "pages"), ({"page": 0}, "pages"),
                            ({"columns": 1 << 23}, "MAX_SERVING_KEYS"), ({"window": -1}, "window"),
                            ({"sinks": -1}, "sinks"), ({"scale": float("inf")}, "finite"), ({"slots": 1}, "fewer"),
                            ({"size": 8}, "workspace too small")):
        assert paged(**change) == bad, change
        assert message in _native.last_error(), (change, _native.last_error())
    size = ctypes.c_int64()
    assert lib.flux_window_attention_workspace_bytes(1, 6, 2, 5, 16, 100, 10, 0, ctypes.byref(size)) == 0
    assert size.value == 0
    assert lib.flux_window_attention_workspace_bytes(1, 6, 2, 1, 16, 100, 10, 0, ctypes.byref(size)) == 0
    assert size.value > 0
    assert lib.flux_window_attention(0, some, some, some, None, None, some, None, 0, 1.0, 1, 6, 2, 1, 100, 16, 10, 0, four,
                                     three, three, None) == bad and "workspace" in _native.last_error()
    assert lib.flux_page_reserve(_books_struct(columns=1 << 23), some, None, 2, some, some, some, 100, None) == bad
    assert lib.flux_page_reserve(_books_struct(), some, None, 0, some, some, some, 100, None) == bad
    assert lib.flux_page_reserve(_books_struct(), some, None, 2, some, some, some, 7, None) == bad
    assert "workspace" in _native.last_error()
    assert lib.flux_page_write(_pool_struct(layers=2), some, some, three, three, 1, 1, some, 4, 2, 4, some, some, None,
                               None) == bad and "one layer" in _native.last_error()
    assert lib.flux_page_copy(_pool_struct(dtype=7), some, some, 1, some, None) == bad
    assert lib.flux_page_copy(_pool_struct(head_dim=0), some, some, 1, some, None) == bad
    assert lib.flux_page_fork(_pool_struct(), _books_struct(pages=5), some, some, 1, some, some, 100, None) == bad
    assert "differ" in _native.last_error()
    assert lib.flux_page_free(_books_struct(refcounts=None), some, 1, some, None) == bad
    assert lib.flux_page_compact(_pool_struct(), _books_struct(), some, some, some, 3, None) == bad
    assert lib.flux_logits_process(0, some, 10, some, some, 2, 0, None, 0, 0, None, None, None, None, None, 0, None, 0,
                                   None, 0, None) == bad
    assert lib.flux_logits_process(0, some, 100000, some, some, 2, 100000, None, 0, 0, None, None, None, None, None, 0,
                                   None, 0, None, 0, None) == bad and "workspace" in _native.last_error()


def test_c_entries_refuse_lists_inside_the_books():
    """Each kernel reads its lists again after it has changed the books."""
    lib, bad = _native.load(), _native.FLUX_ERROR_INVALID_VALUE
    at = {"page_table": 0x10000, "lengths": 0x20000, "refcounts": 0x30000}
    books, some, apart = _books_struct(**at), ctypes.c_void_p(16), ctypes.c_void_p(0x40000)
    sizes = {"page_table": 2 * 4 * 4, "lengths": 2 * 8, "refcounts": 4 * 4}
    for name, start in at.items():
        for inside in (start - 8, start, start + sizes[name] - 1):  # two requests: 16 bytes
            where = ctypes.c_void_p(inside)
            for slots, counts in ((where, None), (where, apart), (apart, where)):
                assert lib.flux_page_reserve(books, slots, counts, 2, some, some, some, 100, None) == bad
                assert "must not lie in the books" in _native.last_error()
            assert lib.flux_page_free(books, where, 2, some, None) == bad
            assert "must not lie in the books" in _native.last_error()
            for parents, children in ((where, apart), (apart, where)):
                assert lib.flux_page_fork(_pool_struct(), books, parents, children, 2, some, some, 100, None) == bad
                assert "must not lie in the books" in _native.last_error()


def test_c_entries_refuse_pages_that_share_memory():
    """Every entry that writes pages, on addresses that nothing reads: the sides are in order in none of the calls."""
    lib, bad, some = _native.load(), _native.FLUX_ERROR_INVALID_VALUE, ctypes.c_void_p(16)

    def pool(key, value):
        layers, pages, heads, rows, dim = key.shape
        out = _native.PagePool(key=0x100000 + 4 * key.storage_offset(), value=0x100000 + 4 * value.storage_offset(),
                               layers=layers, pages=pages, heads=heads, page_size=rows, head_dim=dim, dtype=0)
        out.key_strides[:], out.value_strides[:] = key.stride()[:4], value.stride()[:4]
        return ctypes.byref(out)

    three = (ctypes.c_int64 * 3)(64, 32, 8)

    def message_of(key, value):
        p, found = pool(key, value), set()
        books = _books_struct(pages=key.shape[1], page_size=key.shape[3], page_table=0x10000, lengths=0x20000, refcounts=0x30000)
        calls = [lambda: lib.flux_page_copy(p, some, some, 1, some, None),
                 lambda: lib.flux_page_fork(p, books, some, some, 1, some, some, 1000, None),
                 lambda: lib.flux_page_compact(p, books, some, some, some, 1000, None)]
        if key.shape[0] == 1:
            calls.append(lambda: lib.flux_page_write(p, some, some, three, three, 1, 1, some, 4, 2, 4, some, some, None, None))
        for call in calls:
            assert call() == bad
            found.add(_native.last_error().split(": ")[1])
        assert len(found) == 1
        return found.pop()

    for shape in ((2, 7, 2, 4, 8), (1, 7, 2, 4, 8), (1, 1, 3, 5, 1), (2, 3, 1, 1, 4)):
        for what, key, value, _ in _side_views(shape):
            if key.stride(4) != 1 or value.stride(4) != 1 or not _shares_memory(key, value):
                continue
            assert message_of(key, value) == "key and value pages must not overlap", (shape, what)
    key = torch.zeros(4000)[:448].view(1, 7, 2, 4, 8)
    for strides in ((448, 63, 32, 8, 1), (448, 64, 31, 8, 1), (448, 64, 32, 7, 1), (448, 0, 32, 8, 1)):
        assert message_of(key, torch.zeros(4000).as_strided(key.shape, strides, 1000)) == \
            "key and value pages must not overlap themselves"


def test_c_entries_refuse_table_rows_that_overlap():
    """Requests of different slots write their rows at the same time."""
    lib, bad, some = _native.load(), _native.FLUX_ERROR_INVALID_VALUE, ctypes.c_void_p(16)
    pool = _pool_struct(key=0x100000, value=0x200000)
    for stride in (0, 1, 3):
        books = _books_struct(table_stride=stride, page_table=0x10000, lengths=0x20000, refcounts=0x30000)
        for call in (lambda: lib.flux_page_reserve(books, some, None, 2, some, some, some, 100, None),
                     lambda: lib.flux_page_free(books, some, 2, some, None),
                     lambda: lib.flux_page_fork(pool, books, some, some, 1, some, some, 100, None),
                     lambda: lib.flux_page_compact(pool, books, some, some, some, 100, None)):
            assert call() == bad
            assert "rows must not overlap" in _native.last_error()
    # One row overlaps nothing: the next check answers.
    books = _books_struct(slots=1, table_stride=0, page_table=0x10000, lengths=0x20000, refcounts=0x30000)
    assert lib.flux_page_reserve(books, some, None, 2, some, some, some, 3, None) == bad
    assert "workspace too small" in _native.last_error()


def _header_fields(name):
    """(field, bytes) of a structure in include/flux_amd.h, in their order."""
    text = open(os.path.join(ROOT, "include", "flux_amd.h")).read()
    body = re.search(r"typedef struct \{([^}]*)\} %s;" % name, text).group(1)
    fields = []
    for declaration in filter(None, (d.strip() for d in body.split(";"))):
        kind, field, count = re.fullmatch(r"(int64_t|\w+\*) ?(\w+)(?:\[(\d+)\])?", declaration.replace(" *", "*")).groups()
        fields.append((field, 8 * int(count or 1)))
    return fields


def test_packed_structures_are_those_of_the_header():
    """The operators pack flux_page_books and flux_page_pool into bytes: field by field the header's and ctypes' structures."""
    for name, struct_type in (("flux_page_books", _native.PageBooks), ("flux_page_pool", _native.PagePool)):
        assert _header_fields(name) == [(field, ctypes.sizeof(kind)) for field, kind in struct_type._fields_]
        assert ctypes.sizeof(struct_type) == sum(size for _, size in _header_fields(name))

    table = torch.zeros(5, 9, dtype=i32)[1:4, 2:6]
    lengths, refcounts = torch.zeros(3, dtype=i64), torch.zeros(7, dtype=i32)
    books = _native.PageBooks(page_table=table.data_ptr(), table_stride=9, slots=3, columns=4, lengths=lengths.data_ptr(),
                              refcounts=refcounts.data_ptr(), pages=7, page_size=16)
    assert serving._books(table, lengths, refcounts, 16) == bytes(books)
    books.lengths = None
    assert serving._books(table, None, refcounts, 16) == bytes(books)

    for dtype, code in ((torch.float32, 0), (torch.float16, 1), (torch.bfloat16, 2)):
        key, value = torch.zeros(2, 7, 3, 4, 8, dtype=dtype), torch.zeros(2, 7, 4, 3, 8, dtype=dtype).transpose(2, 3)
        for layered in (True, False):
            pool = _native.PagePool(key=key.data_ptr(), value=value.data_ptr(), layers=2 if layered else 1, pages=7, heads=3,
                                    page_size=4, head_dim=8, dtype=code)
            pool.key_strides[:] = (672 if layered else 0, 96, 32, 8)
            pool.value_strides[:] = (672 if layered else 0, 96, 8, 24)
            assert serving._pool(*((key, value) if layered else (key[0], value[0]))) == bytes(pool)


# --------------------------------------------------------------------------- the plain page model

def test_page_model_keeps_every_sequence():
    """Reserve, write, fork, free and compact in random order: each sequence still reads the tokens it was given."""
    rng = random.Random(5)
    page_size, slots, columns = 3, 6, 5
    model = ref.Pages(1, 16, 1, page_size, 2, slots, columns)
    tokens = {s: [] for s in range(slots)}
    stamp = 0.0
    for _ in range(400):
        action = rng.choice(("grow", "grow", "fork", "free", "compact"))
        if action == "grow":
            named = rng.sample(range(slots), 2)
            counts = [rng.randint(0, 4) for _ in named]
            rows = torch.arange(8.0).view(2, 1, 4, 1).expand(2, 1, 4, 2) + stamp
            stamp += 8
            positions, _ = model.reserve(named, counts)
            model.write(0, rows, -rows, named, positions, counts)
            for i, slot in enumerate(named):
                if positions[i] >= 0:
                    tokens[slot] += rows[i, 0, : counts[i], 0].tolist()
        elif action == "fork":
            parent, child = rng.sample(range(slots), 2)
            if model.fork([parent], [child]) == [ref.DONE]:
                tokens[child] = list(tokens[parent])
        elif action == "free":
            slot = rng.randrange(slots)
            model.free([slot])
            tokens[slot] = []
        else:
            model.compact()
        for slot in range(slots):
            assert model.lengths[slot] == len(tokens[slot])
            read = [float(model.key[0, model.table[slot][j // page_size], 0, j % page_size, 0])
                    for j in range(len(tokens[slot]))]
            assert read == tokens[slot]
        held = [0] * model.pages
        for row in model.table:
            for p in row:
                if p >= 0:
                    held[p] += 1
        assert held == model.refcounts
