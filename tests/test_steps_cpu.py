"""Operators of mixed steps without a GPU: schemas, refusals with their messages, FakeTensor shapes, C entries' checks."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from flux_amd import _native, ops
from flux_amd.ops import steps

i64, i32, f32 = torch.int64, torch.int32, torch.float32


def _chunk(tokens=7, heads=6, kv_heads=2, dim=16, pages=5, page_size=4, slots=3, columns=3, requests=2, dtype=f32):
    return {"query": torch.zeros(tokens, heads, dim, dtype=dtype),
            "key_pages": torch.zeros(pages, kv_heads, page_size, dim, dtype=dtype),
            "value_pages": torch.zeros(pages, kv_heads, page_size, dim, dtype=dtype),
            "page_table": torch.zeros(slots, columns, dtype=i32), "lengths": torch.ones(slots, dtype=i64),
            "offsets": torch.arange(requests + 1), "scale": 0.25}


def _rows(tokens=3, kv_heads=2, dim=8, pages=7, page_size=4):
    shape = (pages, kv_heads, page_size, dim)
    return {"key": torch.zeros(tokens, kv_heads, dim), "value": torch.zeros(tokens, kv_heads, dim),
            "key_pages": torch.zeros(shape), "value_pages": torch.zeros(shape), "rows": torch.arange(tokens)}


CALLS = {
    "paged_step_layout": lambda: {"page_table": torch.zeros(3, 4, dtype=i32), "slots": torch.arange(2), "positions": torch.arange(2),
                                  "counts": torch.ones(2, dtype=i64), "page_size": 4, "tokens": 9},
    "paged_cache_write_rows": _rows,
    "paged_chunk_attention": _chunk,
    "logits_sample": lambda: {"logits": torch.zeros(2, 100), "uniforms": torch.zeros(2)},
}


def test_every_operator_is_registered_and_exported():
    assert set(CALLS) == set(ops.STEP_OPERATOR_NAMES) == set(steps.STEP_SCHEMAS)
    for name in ops.STEP_OPERATOR_NAMES:
        assert hasattr(torch.ops.flux, name)
        assert f"{name}_native" in ops.__all__ and callable(getattr(ops, f"{name}_native"))
    assert ops.native_paged_step_is_available() and ops.native_logits_sample_is_available()


@pytest.mark.parametrize("name", sorted(CALLS))
def test_valid_cpu_tensors_are_refused_for_want_of_a_kernel(name):
    with pytest.raises(RuntimeError, match="no CPU kernel"):
        getattr(torch.ops.flux, name)(**CALLS[name]())
    with pytest.raises(RuntimeError, match="no CPU kernel"):
        getattr(ops, f"{name}_native")(**CALLS[name]())


_store = torch.zeros(7 * 2 * 4 * 8 + 48)
REFUSED = [
    ("paged_step_layout", {"page_table": torch.zeros(3, 4, dtype=i64)}, "page_table must be int32"),
    ("paged_step_layout", {"page_table": torch.zeros(4, 3, dtype=i32).t()}, "rows must be contiguous"),
    ("paged_step_layout", {"page_size": 0}, "page_size must be positive"),
    ("paged_step_layout", {"page_size": 1 << 23}, "at most 16777216"),
    ("paged_step_layout", {"tokens": -1}, "tokens must be within"),
    ("paged_step_layout", {"tokens": (1 << 24) + 1}, "tokens must be within"),
    ("paged_step_layout", {"slots": torch.arange(2, dtype=i32)}, "slots must be a contiguous int64"),
    ("paged_step_layout", {"slots": torch.arange(4)[::2]}, "slots must be a contiguous int64"),
    ("paged_step_layout", {"slots": torch.zeros(65536, dtype=i64)}, "more than 65535 requests"),
    ("paged_step_layout", {"positions": torch.arange(3)}, "positions must have one entry"),
    ("paged_step_layout", {"counts": torch.arange(3)}, "counts must have one entry"),
    ("paged_step_layout", {"counts": torch.zeros(2)}, "counts must be a contiguous int64"),
    ("paged_cache_write_rows", {"key": torch.zeros(3, 2, 1, 8)}, r"key and value must be \[tokens"),
    ("paged_cache_write_rows", {"value": torch.zeros(2, 2, 8)}, "of one shape"),
    ("paged_cache_write_rows", {"key": torch.zeros(3, 2, 8, dtype=torch.float16)}, "the pages' dtype"),
    ("paged_cache_write_rows", {"key": torch.zeros(3, 1, 8), "value": torch.zeros(3, 1, 8)}, "heads and head dimension"),
    ("paged_cache_write_rows", {"key": torch.zeros(3, 8, 2).transpose(1, 2)}, "unit stride"),
    ("paged_cache_write_rows", {"rows": torch.arange(2)}, "rows must have one entry"),
    ("paged_cache_write_rows", {"rows": torch.arange(3, dtype=i32)}, "rows must be a contiguous int64"),
    ("paged_cache_write_rows", {"key_pages": torch.zeros(2, 7, 2, 4, 8), "value_pages": torch.zeros(2, 7, 2, 4, 8)},
     r"must be \[pages, kv_heads"),
    ("paged_cache_write_rows", {"key_pages": torch.zeros(1, 2, 4, 8).expand(7, 2, 4, 8)}, "must not overlap itself"),
    ("paged_cache_write_rows", {"key_pages": _store[:448].view(7, 2, 4, 8), "value_pages": _store[8:456].view(7, 2, 4, 8)},
     "key and value pages must not overlap"),
    ("paged_cache_write_rows", {"key_pages": _store[48:].view(7, 2, 4, 8), "key": _store[:48].view(3, 2, 8)}, "must not alias"),
    ("paged_cache_write_rows", {"key": torch.zeros(3, 2, 8, requires_grad=True)}, "inference-only"),
    ("paged_chunk_attention", {"query": torch.zeros(7, 6, 1, 16)}, r"query must be \[tokens"),
    ("paged_chunk_attention", {"query": torch.zeros(7, 6, 16, dtype=torch.float64)}, "share dtype"),
    ("paged_chunk_attention", {"value_pages": torch.zeros(5, 2, 4, 16, dtype=torch.float16)}, "share dtype"),
    ("paged_chunk_attention", {"value_pages": torch.zeros(5, 2, 3, 16)}, "page shapes must match"),
    ("paged_chunk_attention", {"query": torch.zeros(7, 0, 16)}, "non-empty"),
    ("paged_chunk_attention", {"query": torch.zeros(7, 6, 8)}, "head dimensions must match"),
    ("paged_chunk_attention", {**_chunk(dim=257)}, "at most 256"),
    ("paged_chunk_attention", {"query": torch.zeros(7, 5, 16)}, "divisible by KV heads"),
    ("paged_chunk_attention", {"query": torch.zeros(1, 1, 16).expand((1 << 24) + 1, 2, 16)}, "more than 16777216 tokens"),
    ("paged_chunk_attention", {"query": torch.zeros(1, 1, 16).expand(1 << 24, 18, 16)}, "rows of a KV head"),
    ("paged_chunk_attention", {"page_table": torch.zeros(3, 3, dtype=i64)}, "page_table must be int32"),
    ("paged_chunk_attention", {"page_table": torch.zeros(3, 3, dtype=i32).t()}, "rows must be contiguous"),
    ("paged_chunk_attention", {"page_table": torch.zeros(3, 1, dtype=i32).expand(3, 5000000)}, "must be contiguous|16777216"),
    ("paged_chunk_attention", {"lengths": torch.ones(2, dtype=i64)}, "one entry per page_table row"),
    ("paged_chunk_attention", {"lengths": torch.ones(3, dtype=i32)}, "lengths must be a contiguous int64"),
    ("paged_chunk_attention", {"offsets": torch.zeros(0, dtype=i64)}, "one entry more than the requests"),
    ("paged_chunk_attention", {"offsets": torch.zeros(65537, dtype=i64)}, "at most 65535"),
    ("paged_chunk_attention", {"offsets": torch.zeros(3, dtype=i32)}, "offsets must be a contiguous int64"),
    ("paged_chunk_attention", {"offsets": torch.zeros(5, dtype=i64)}, "without slots"),
    ("paged_chunk_attention", {"slots": torch.zeros(3, dtype=i64)}, "slots must have one entry per request"),
    ("paged_chunk_attention", {"positions": torch.zeros(2, dtype=i32)}, "positions must be a contiguous int64"),
    ("paged_chunk_attention", {"key_pages": torch.zeros(5, 2, 16, 4).transpose(2, 3)}, "unit stride"),
    ("paged_chunk_attention", {"window": -1}, "window and sinks"),
    ("paged_chunk_attention", {"sinks": (1 << 24) + 1}, "window and sinks"),
    ("paged_chunk_attention", {"scale": float("nan")}, "finite FP32"),
    ("paged_chunk_attention", {"scale": 1e39}, "finite FP32"),
    ("paged_chunk_attention", {"query": torch.zeros(7, 6, 16, requires_grad=True)}, "inference-only"),
    ("logits_sample", {"logits": torch.zeros(100)}, r"logits must be \[rows, vocab\]"),
    ("logits_sample", {"logits": torch.zeros(2, 0)}, "non-empty"),
    ("logits_sample", {"logits": torch.zeros(1, 1).expand(2, (1 << 24) + 1)}, "at most 16777216"),
    ("logits_sample", {"logits": torch.zeros(2, 100, dtype=torch.float64)}, "dtype float32"),
    ("logits_sample", {"logits": torch.zeros(100, 2).t()}, "rows must be contiguous"),
    ("logits_sample", {"uniforms": torch.zeros(3)}, "uniforms must be a contiguous float32"),
    ("logits_sample", {"uniforms": torch.zeros(2, dtype=torch.float64)}, "uniforms must be a contiguous float32"),
    ("logits_sample", {"temperature": torch.zeros(4)[::2]}, "temperature must be a contiguous float32"),
    ("logits_sample", {"top_k": torch.zeros(2, dtype=i32)}, "top_k must be a contiguous int64"),
    ("logits_sample", {"top_p": torch.zeros(1)}, "top_p must be a contiguous float32"),
    ("logits_sample", {"min_p": torch.zeros(2, 1)}, "min_p must be a contiguous float32"),
    ("logits_sample", {"logits": torch.zeros(2, 100, requires_grad=True)}, "inference-only"),
]


@pytest.mark.parametrize("name,change,message", REFUSED)
def test_refusals(name, change, message):
    with pytest.raises(RuntimeError, match=message):
        getattr(torch.ops.flux, name)(**{**CALLS[name](), **change})


@pytest.mark.parametrize("name,change,message", [r for r in REFUSED if "requires_grad" not in str(r[1]) and "alias" not in r[2] and
                                                 "key and value pages" not in r[2]][::3])
def test_fake_tensors_are_refused_alike(name, change, message):
    mode = FakeTensorMode()
    args = {k: mode.from_tensor(v) if isinstance(v, torch.Tensor) else v for k, v in {**CALLS[name](), **change}.items()}
    with mode, pytest.raises(RuntimeError, match=message):
        getattr(torch.ops.flux, name)(**args)


def test_fake_shapes():
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        def fake(name, **change):
            return {k: mode.from_tensor(v) if isinstance(v, torch.Tensor) else v for k, v in {**CALLS[name](), **change}.items()}

        offsets, request, position, rows = torch.ops.flux.paged_step_layout(**fake("paged_step_layout"))
        assert offsets.shape == (3,) and request.shape == position.shape == rows.shape == (9,) and rows.dtype == i64
        assert torch.ops.flux.paged_cache_write_rows(**fake("paged_cache_write_rows")) is None
        out = torch.ops.flux.paged_chunk_attention(**fake("paged_chunk_attention", **_chunk(dtype=torch.bfloat16)))
        assert out.shape == (7, 6, 16) and out.dtype == torch.bfloat16
        tokens, probabilities = torch.ops.flux.logits_sample(**fake("logits_sample"))
        assert tokens.shape == probabilities.shape == (2,) and tokens.dtype == i64 and probabilities.dtype == f32


def test_c_entries_refuse_before_any_launch():
    lib, some = _native.load(), ctypes.c_void_p(16)  # never dereferenced
    bad = _native.FLUX_ERROR_INVALID_VALUE
    three, two = (ctypes.c_int64 * 3)(64, 16, 1), (ctypes.c_int64 * 2)(64, 16)
    minus = (ctypes.c_int64 * 3)(64, -16, 1)

    def chunk(dtype=0, query=some, table=some, lengths=some, offsets=some, output=some, workspace=some, size=1 << 30, scale=1.0,
              tokens=7, requests=2, heads=6, kv=2, dim=16, pages=4, page=4, slots=2, columns=400, stride=400, window=0, sinks=0,
              strides=three):
        return lib.flux_paged_chunk_attention(dtype, query, some, some, table, lengths, offsets, None, None, output, workspace, size,
                                              scale, tokens, requests, heads, kv, dim, pages, page, slots, columns, stride, window,
                                              sinks, strides, three, three, None)

    for change, message in (({"query": None}, "null"), ({"table": None}, "null"), ({"lengths": None}, "null"),
                            ({"offsets": None}, "null"), ({"output": None}, "null"), ({"strides": None}, "null"),
                            ({"dtype": 3}, "dtype"), ({"tokens": 0}, "shape"), ({"tokens": (1 << 24) + 1}, "shape"),
                            ({"requests": 0}, "shape"), ({"requests": 65536}, "shape"), ({"heads": 5}, "shape"),
                            ({"dim": 257}, "shape"), ({"tokens": 1 << 24, "heads": 18}, "shape"), ({"pages": 0}, "pages"),
                            ({"page": 0}, "pages"), ({"columns": 1 << 23}, "MAX_SERVING_KEYS"), ({"window": -1}, "window"),
                            ({"sinks": -1}, "sinks"), ({"scale": float("inf")}, "finite"), ({"slots": 1}, "fewer"),
                            ({"strides": minus}, "negative"), ({"stride": -1}, "negative"), ({"size": 8}, "workspace"),
                            ({"workspace": None}, "workspace"), ({"workspace": ctypes.c_void_p(20)}, "16-byte")):
        assert chunk(**change) == bad, change
        assert message in _native.last_error(), (change, _native.last_error())
    size = ctypes.c_int64()
    # A row of the table holds too few keys for tiles to be cut: no workspace.
    assert lib.flux_paged_chunk_attention_workspace_bytes(0, 7, 2, 6, 2, 16, 4, 3, 0, 0, ctypes.byref(size)) == 0 and size.value == 0
    for dtype in range(3):
        assert lib.flux_paged_chunk_attention_workspace_bytes(dtype, 7, 2, 6, 2, 16, 4, 4000, 0, 0, ctypes.byref(size)) == 0
        assert size.value > 0
    assert lib.flux_paged_chunk_attention_workspace_bytes(0, 0, 2, 6, 2, 16, 4, 4000, 0, 0, ctypes.byref(size)) == bad

    def layout(table=some, page=4, slots=2, columns=4, stride=4, requests=2, tokens=9, rows=some):
        return lib.flux_step_layout(table, stride, slots, columns, page, some, some, None, requests, tokens, some, some, some, rows, None)

    for change, message in (({"table": None}, "null"), ({"rows": None}, "null"), ({"page": 0}, "shape"), ({"columns": 1 << 23}, "shape"),
                            ({"stride": -1}, "shape"), ({"requests": 0}, "shape"), ({"requests": 65536}, "shape"),
                            ({"tokens": 0}, "shape"), ({"tokens": (1 << 24) + 1}, "shape"), ({"slots": 0}, "shape")):
        assert layout(**change) == bad, change
        assert message in _native.last_error(), change

    def pool(value=0x200000, layers=1):
        out = _native.PagePool(key=0x100000, value=value, layers=layers, pages=4, heads=2, page_size=4, head_dim=8, dtype=0)
        out.key_strides[:] = out.value_strides[:] = (256, 64, 32, 8)
        return ctypes.byref(out)

    for args, message in (((pool(), None, some, two, two, 3, some), "null"), ((pool(), some, some, two, two, 0, some), "shape"),
                          ((pool(layers=2), some, some, two, two, 3, some), "one layer"),
                          ((pool(value=0x100010), some, some, two, two, 3, some), "must not overlap"),
                          ((pool(), some, some, minus, two, 3, some), "negative"), ((pool(), some, some, two, two, 3, None), "null")):
        assert lib.flux_page_write_rows(*args, None) == bad
        assert message in _native.last_error(), message

    def sample(dtype=0, logits=some, stride=100, uniforms=some, rows=2, vocab=100, tokens=some, shares=some):
        return lib.flux_logits_sample(dtype, logits, stride, uniforms, None, None, None, None, tokens, shares, rows, vocab, None, 0, None)

    for change, message in (({"logits": None}, "null"), ({"uniforms": None}, "null"), ({"tokens": None}, "null"),
                            ({"shares": None}, "null"), ({"dtype": -1}, "dtype"), ({"rows": 0}, "shape"), ({"vocab": 0}, "shape"),
                            ({"vocab": (1 << 24) + 1}, "shape"), ({"rows": 1 << 20, "vocab": 1 << 20}, "shape"),
                            ({"stride": -1}, "shape")):
        assert sample(**change) == bad, change
        assert message in _native.last_error(), change
    assert lib.flux_logits_sample_workspace_bytes(2, 128000, ctypes.byref(size)) == 0
    assert lib.flux_logits_sample_workspace_bytes(0, 100, ctypes.byref(size)) == bad


def _sample_meta(rows, vocab):
    return {"logits": torch.empty(rows, vocab), "uniforms": torch.empty(rows)}


@pytest.mark.parametrize("rows,vocab", [((1 << 20) + 1, 8), (1 << 20, 1 << 13), (1 << 9, 1 << 24)])
def test_sampling_beyond_the_c_entries_limits_is_refused_by_every_layer(rows, vocab):
    with FakeTensorMode(), pytest.raises(RuntimeError, match="more than 1048576 rows"):
        torch.ops.flux.logits_sample(**_sample_meta(rows, vocab))
    logits = torch.zeros(vocab).expand(rows, vocab)
    with pytest.raises(RuntimeError, match="more than 1048576 rows"):
        torch.ops.flux.logits_sample(logits, torch.zeros(rows))
    size = ctypes.c_int64()
    assert _native.load().flux_logits_sample_workspace_bytes(rows, vocab, ctypes.byref(size)) == _native.FLUX_ERROR_INVALID_VALUE


def test_sampling_no_rows_is_a_valid_call():
    with FakeTensorMode():
        tokens, probabilities = torch.ops.flux.logits_sample(**_sample_meta(0, 100))
    assert tokens.shape == probabilities.shape == (0,) and tokens.dtype == i64 and probabilities.dtype == f32
    with pytest.raises(RuntimeError, match="no CPU kernel"):
        torch.ops.flux.logits_sample(torch.zeros(0, 100), torch.zeros(0))


def _fake_chunk(tokens, heads, kv_heads, dim, requests=1, pages=5, dtype=torch.bfloat16):
    return {"query": torch.empty(tokens, heads, dim, dtype=dtype), "key_pages": torch.empty(pages, kv_heads, 4, dim, dtype=dtype),
            "value_pages": torch.empty(pages, kv_heads, 4, dim, dtype=dtype), "page_table": torch.empty(requests, 3, dtype=i32),
            "lengths": torch.empty(requests, dtype=i64), "offsets": torch.empty(requests + 1, dtype=i64), "scale": 0.25}


def _refused_by_c(dtype, tokens, heads, kv_heads, dim, requests=1, columns=4000):
    size = ctypes.c_int64()
    return _native.load().flux_paged_chunk_attention_workspace_bytes(dtype, tokens, requests, heads, kv_heads, dim, 4, columns, 0, 0,
                                                                     ctypes.byref(size)) != 0


@pytest.mark.parametrize("sizes,message", [((1, 65536, 65536, 16), "more than 65535 query heads"),
                                           ((1, 65535, 65535, 16), None),
                                           ((1 << 24, 128, 128, 128), "tiles are 16777216 or more"),
                                           ((1 << 23, 128, 128, 128), None)])
def test_chunk_sizes_beyond_the_c_entries_limits_are_refused_by_every_layer(sizes, message):
    with FakeTensorMode():
        if message:
            with pytest.raises(RuntimeError, match=message):
                torch.ops.flux.paged_chunk_attention(**_fake_chunk(*sizes))
        else:
            assert torch.ops.flux.paged_chunk_attention(**_fake_chunk(*sizes)).shape == (sizes[0], sizes[1], sizes[3])
        with pytest.raises(RuntimeError, match="268435456 pages"):
            torch.ops.flux.paged_chunk_attention(**_fake_chunk(1, 1, 1, 16, pages=(1 << 28) + 1))
    assert _refused_by_c(2, *sizes) == (message is not None)
    lib, three = _native.load(), (ctypes.c_int64 * 3)(64, 16, 1)
    some = ctypes.c_void_p(16)  # never dereferenced
    if message and "tiles" in message:
        assert lib.flux_paged_chunk_attention(2, some, some, some, some, some, some, None, None, some, some, 1 << 40, 1.0, sizes[0], 1,
                                              *sizes[1:], 4, 4, 2, 400, 400, 0, 0, three, three, three, None) == _native.FLUX_ERROR_INVALID_VALUE
        assert "tiles" in _native.last_error()


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_what_the_c_entry_refuses_for_its_tiles_is_refused_before(dtype):
    of = {0: f32, 1: torch.float16, 2: torch.bfloat16}[dtype]
    refused = 0
    for heads, kv_heads in ((1, 1), (7, 7), (128, 128), (128, 16), (1000, 1000), (8192, 8192), (65535, 65535)):
        for dim in (16, 64, 65, 128, 129):
            for requests in (1, 3000, 65535):
                for tokens in (1, 3, 255, 2048, 65535, 1 << 20, 1 << 21, 1 << 22, 1 << 23, (1 << 24) - 1):
                    if tokens * (heads // kv_heads) > 1 << 27 or not _refused_by_c(dtype, tokens, heads, kv_heads, dim, requests):
                        continue
                    refused += 1
                    assert steps._workgroups((tokens, heads, dim), kv_heads, of, requests) >= 1 << 24
                    assert tokens * heads + 16 * ((requests + 64) * kv_heads + 1024) >= 1 << 28
    assert refused > 20


@pytest.mark.parametrize("shape", [((1 << 28) + 1, 1, 1, 1), (1, 1, (1 << 24) + 1, 1), (1, (1 << 20) + 1, 1, 1), (1, 1, 1, (1 << 20) + 1),
                                   (1, 1 << 13, 1, (1 << 11) + 1), (1, 1 << 10, 1 << 10, 257)])
def test_row_writes_beyond_the_c_entries_limits_are_refused_by_every_layer(shape):
    with FakeTensorMode(), pytest.raises(RuntimeError, match="more than 268435456 pages or elements a page"):
        torch.ops.flux.paged_cache_write_rows(torch.empty(2, shape[1], shape[3]), torch.empty(2, shape[1], shape[3]), torch.empty(shape),
                                              torch.empty(shape), torch.empty(2, dtype=i64))
    pool = _native.PagePool(key=1 << 32, value=1 << 60, layers=1, pages=shape[0], heads=shape[1], page_size=shape[2], head_dim=shape[3], dtype=0)
    pool.key_strides[:] = pool.value_strides[:] = (0, shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3])
    two, some = (ctypes.c_int64 * 2)(shape[1] * shape[3], shape[3]), ctypes.c_void_p(16)
    assert _native.load().flux_page_write_rows(ctypes.byref(pool), some, some, two, two, 2, some, None) == _native.FLUX_ERROR_INVALID_VALUE
    assert "shape" in _native.last_error()


def test_sampling_refuses_a_workspace_that_its_atomics_cannot_use():
    lib, size, some = _native.load(), ctypes.c_int64(), ctypes.c_void_p(16)  # never dereferenced
    assert lib.flux_logits_sample_workspace_bytes(2, 128000, ctypes.byref(size)) == 0 and size.value > 0
    for workspace, given in ((None, size.value), (ctypes.c_void_p(64), size.value - 1), (ctypes.c_void_p(68), size.value),
                             (ctypes.c_void_p(72), size.value)):
        assert lib.flux_logits_sample(0, some, 128000, some, None, None, None, None, some, some, 2, 128000, workspace, given,
                                      None) == _native.FLUX_ERROR_INVALID_VALUE
        assert "16-byte aligned" in _native.last_error()
