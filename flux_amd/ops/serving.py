"""``torch.ops.flux.*`` for serving several sequences: attention over a paged K/V cache, windowed attention, the pages
themselves, and logits on their way to the next token.

They stand next to the one-sequence operators of ``flux_amd.ops.native`` and follow their manner: arguments are
checked on the host, each ROCm kernel is a call through the C ABI of ``libflux_amd.so`` on the tensors' current stream,
CPU tensors are checked and then refused, FakeTensor contracts are registered, and everything is inference-only.
Nothing here synchronises with the GPU: lengths, tables and lists stay on the device, and what a request of a page
operator came to is in the status it returns.

A cache in pages is ``key_pages`` and ``value_pages`` ``[pages, kv_heads, page_size, head_dim]`` of one layer, or with
a leading layer dimension for the operators that move pages, and the books that all layers share: ``page_table`` int32
``[slots, columns]`` (-1: no page), ``lengths`` int64 ``[slots]`` and ``refcounts`` int32 ``[pages]`` (0: free).
"""

from __future__ import annotations

import ctypes
import functools
import math
import struct

import torch

from flux_amd import _native
from flux_amd.ops.native import (_LIBRARY, _aliases, _availability, _check, _cpu_kernel, _finite_fp32, _grad_free,
                                 _require_gpu, _require_library)

PAGE_DONE, PAGE_OUT_OF_RANGE, PAGE_REPEATED, PAGE_NO_ROOM, PAGE_OCCUPIED = range(5)

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_MAX_DIM = 256
_MAX_KEYS = 1 << 24  # positions of one sequence
_MAX_VOCAB = 1 << 24

SERVING_SCHEMAS = {
    "paged_decode_attention": ("paged_decode_attention(Tensor query, Tensor key_pages, Tensor value_pages, "
                               "Tensor page_table, Tensor lengths, float scale, int window=0, int sinks=0, "
                               "Tensor? slots=None) -> Tensor"),
    "paged_decode_attention_out": ("paged_decode_attention_out(Tensor query, Tensor key_pages, Tensor value_pages, "
                                   "Tensor page_table, Tensor lengths, float scale, int window, int sinks, "
                                   "Tensor? slots, Tensor(a!) output, Tensor(b!) workspace) -> Tensor(a!)"),
    "window_attention": ("window_attention(Tensor query, Tensor key, Tensor value, float scale, int window, "
                         "int sinks=0, Tensor? lengths=None, Tensor? starts=None) -> Tensor"),
    "paged_cache_reserve": ("paged_cache_reserve(Tensor(a!) page_table, Tensor(b!) lengths, Tensor(c!) refcounts, "
                            "int page_size, Tensor slots, Tensor? counts=None) -> (Tensor positions, Tensor status)"),
    "paged_cache_write": ("paged_cache_write(Tensor key, Tensor value, Tensor(a!) key_pages, Tensor(b!) value_pages, "
                          "Tensor page_table, Tensor slots, Tensor positions, Tensor? counts=None) -> ()"),
    "paged_cache_copy": ("paged_cache_copy(Tensor(a!) key_pages, Tensor(b!) value_pages, Tensor source, "
                         "Tensor target) -> Tensor"),
    "paged_cache_fork": ("paged_cache_fork(Tensor(a!) key_pages, Tensor(b!) value_pages, Tensor(c!) page_table, "
                         "Tensor(d!) lengths, Tensor(e!) refcounts, Tensor parents, Tensor children) -> Tensor"),
    "paged_cache_free": ("paged_cache_free(Tensor(a!) page_table, Tensor(b!) lengths, Tensor(c!) refcounts, "
                         "Tensor slots) -> Tensor"),
    "paged_cache_compact": ("paged_cache_compact(Tensor(a!) key_pages, Tensor(b!) value_pages, Tensor(c!) page_table, "
                            "Tensor(d!) refcounts) -> (Tensor page_map, Tensor used)"),
    "logits_process": ("logits_process(Tensor logits, Tensor? history=None, Tensor? history_lengths=None, "
                       "Tensor? repetition=None, Tensor? frequency=None, Tensor? presence=None, Tensor? bias=None, "
                       "Tensor? allowed=None) -> (Tensor processed, Tensor tokens)"),
}

SERVING_OPERATOR_NAMES = tuple(SERVING_SCHEMAS)

for _schema in SERVING_SCHEMAS.values():
    _LIBRARY.define(_schema)

# Checks and arguments are a large part of a small call's time (one sequence of 900 keys: 18.7 us, in a graph 12.5): shapes are
# read once, conditions are tested in place, messages are whole literals, sizes that only depend on shapes come from small
# caches, and structures and strides are packed into bytes (a ctypes array of four costs 0.5 us, its bytes 0.2).
_four = struct.Struct("4q").pack
_page_books = struct.Struct("8q").pack   # flux_page_books
_page_pool = struct.Struct("16q").pack   # flux_page_pool

def _address(tensor):
    return None if tensor is None else tensor.data_ptr()


def _check_list(tensor, dtype, device, message: str, length=None, length_message: str = "") -> None:
    """A contiguous vector of ``dtype`` (and ``length``) on ``device``."""
    shape = tensor.shape
    if not (len(shape) == 1 and tensor.dtype is dtype and tensor.device == device and tensor.is_contiguous()):
        _check(False, message)
    if length is not None:
        _check(shape[0] == length, length_message)


def _call(function: str, *args) -> None:
    status = getattr(_native._lib or _native.load(), function)(*args)
    if status:
        _native.check(status)


def _launch(function: str, device: torch.device, *args) -> None:
    """A C entry on the device's current stream."""
    if device.index == torch.cuda.current_device():
        _call(function, *args, _native.current_stream(device))
    else:
        with torch.cuda.device(device):
            _call(function, *args, _native.current_stream(device))


def _ready(what: str) -> None:
    if _native._lib is None:
        _require_library(what)


@functools.lru_cache(maxsize=1024)
def _size_from(function: str, *sizes) -> int:
    """A workspace size of the C ABI, a function of shapes alone."""
    value = ctypes.c_int64(0)
    _call(function, *sizes, ctypes.byref(value))
    return value.value


# ---------------------------------------------------------------------------
# paged_decode_attention

def _validate_paged(query, key_pages, value_pages, page_table, lengths, scale, window=0, sinks=0, slots=None) -> None:
    shape, pages, table, dtype, device = query.shape, key_pages.shape, page_table.shape, query.dtype, query.device
    if not (len(shape) == 4 and len(pages) == 4 and value_pages.dim() == 4):
        _check(False, "flux::paged_decode_attention: query and pages must be rank four")
    if not (dtype in _TYPES and key_pages.dtype is dtype and value_pages.dtype is dtype):
        _check(False, "flux::paged_decode_attention: query and pages must share dtype float32, float16 or bfloat16")
    if not (shape[2] == 1):
        _check(False, "flux::paged_decode_attention: query length must be one")
    if not (pages == value_pages.shape):
        _check(False, "flux::paged_decode_attention: key and value page shapes must match")
    if not (0 not in shape and 0 not in pages):
        _check(False, "flux::paged_decode_attention: tensor dimensions must be non-empty")
    if not (shape[3] == pages[3] and shape[3] <= _MAX_DIM):
        _check(False, "flux::paged_decode_attention: head dimensions must match and be at most 256")
    if not (shape[1] % pages[1] == 0):
        _check(False, "flux::paged_decode_attention: query heads must be divisible by KV heads")
    if not (len(table) == 2 and page_table.dtype is torch.int32 and table[1] > 0):
        _check(False, "flux::paged_decode_attention: page_table must be int32 [slots, columns]")
    if not (page_table.stride(1) == 1 or table[1] == 1):
        _check(False, "flux::paged_decode_attention: page_table rows must be contiguous")
    if not (table[1] * pages[2] <= _MAX_KEYS):
        _check(False, "flux::paged_decode_attention: page_table holds more than 16777216 positions a row")
    _check_list(lengths, torch.int64, device,
                "flux::paged_decode_attention: lengths must be a contiguous int64 vector on the query device",
                table[0], "flux::paged_decode_attention: lengths must have one entry per page_table row")
    if slots is None:
        _check(table[0] == shape[0],
               "flux::paged_decode_attention: without slots page_table must have one row per sequence")
    else:
        _check_list(slots, torch.int64, device,
                    "flux::paged_decode_attention: slots must be a contiguous int64 vector on the query device",
                    shape[0], "flux::paged_decode_attention: slots must have one entry per sequence")
    if not (key_pages.device == device and value_pages.device == device and page_table.device == device):
        _check(False, "flux::paged_decode_attention: tensor devices must match")
    if not (key_pages.stride(3) == 1 and value_pages.stride(3) == 1 or pages[3] == 1):
        _check(False, "flux::paged_decode_attention: pages must have unit stride along the head dimension")
    if not (0 <= window <= _MAX_KEYS and 0 <= sinks <= _MAX_KEYS):
        _check(False, "flux::paged_decode_attention: window and sinks must be within [0, 16777216]")
    if not (_finite_fp32(scale)):
        _check(False, "flux::paged_decode_attention: scale must be a finite FP32 value")
    if torch.is_grad_enabled():
        _grad_free("flux::paged_decode_attention", query, key_pages, value_pages)


def paged_decode_workspace_bytes(query: torch.Tensor, key_pages: torch.Tensor, page_table: torch.Tensor, window: int = 0,
                                 sinks: int = 0) -> int:
    """Device workspace (bytes) that flux::paged_decode_attention needs for these shapes."""
    shape, pages = query.shape, key_pages.shape
    return _size_from("flux_paged_decode_attention_workspace_bytes", shape[0], shape[1], pages[1], shape[3],
                      page_table.shape[1] * pages[2], window, sinks)


def _launch_paged(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots, output, workspace):
    batch, heads, _, dim = query.shape
    pages, kv_heads, page_size, _ = key_pages.shape
    slot_count, columns = page_table.shape
    _launch("flux_paged_decode_attention", query.device, _TYPES[query.dtype], query.data_ptr(), key_pages.data_ptr(),
            value_pages.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), _address(slots), output.data_ptr(),
            workspace.data_ptr(), workspace.numel() * 4, scale, batch, heads, kv_heads, dim, pages, page_size, slot_count,
            columns, page_table.stride(0), window, sinks, _four(*query.stride()), _four(*key_pages.stride()),
            _four(*value_pages.stride()))


def _paged_cuda(query, key_pages, value_pages, page_table, lengths, scale, window=0, sinks=0, slots=None):
    _validate_paged(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots)
    _check(query.is_cuda, "flux::paged_decode_attention: CUDA dispatch requires CUDA tensors")
    output = query.new_empty(query.shape)
    workspace = lengths.new_empty(paged_decode_workspace_bytes(query, key_pages, page_table, window, sinks) // 4,
                                  dtype=torch.float32)
    _launch_paged(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots, output, workspace)
    return output


def _validate_paged_out(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots, output,
                        workspace) -> None:
    _validate_paged(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots)
    op = "flux::paged_decode_attention_out"
    _check(output.shape == query.shape and output.dtype == query.dtype and output.device == query.device and
           output.is_contiguous(), f"{op}: output must be contiguous, of the query's shape, dtype and device")
    _check(workspace.dtype == torch.float32 and workspace.device == query.device and workspace.is_contiguous(),
           f"{op}: workspace must be contiguous float32 on the query device")


def _validate_paged_out_memory(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots, output,
                               workspace) -> None:
    _validate_paged_out(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots, output,
                        workspace)
    op = "flux::paged_decode_attention_out"
    _check(not _aliases(output, workspace), f"{op}: output and workspace must not alias")
    for tensor in (query, key_pages, value_pages, page_table, lengths, slots):
        _check(tensor is None or not (_aliases(output, tensor) or _aliases(workspace, tensor)),
               f"{op}: output and workspace must not alias an input")


def _paged_out_cuda(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots, output, workspace):
    _validate_paged_out_memory(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots, output,
                               workspace)
    _require_gpu("flux::paged_decode_attention_out", query)
    _check(workspace.numel() * 4 >= paged_decode_workspace_bytes(query, key_pages, page_table, window, sinks),
           "flux::paged_decode_attention_out: workspace is too small (paged_decode_workspace_bytes)")
    _launch_paged(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots, output, workspace)
    return output


# ---------------------------------------------------------------------------
# window_attention

def _validate_window(query, key, value, scale, window, sinks=0, lengths=None, starts=None) -> None:
    shape, keys, dtype, device = query.shape, key.shape, query.dtype, query.device
    if not (len(shape) == 4 and len(keys) == 4 and value.dim() == 4):
        _check(False, "flux::window_attention: query, key and value must be rank four")
    if not (dtype in _TYPES and key.dtype is dtype and value.dtype is dtype):
        _check(False, "flux::window_attention: query, key and value must share dtype float32, float16 or bfloat16")
    if not (keys == value.shape):
        _check(False, "flux::window_attention: key and value shapes must match")
    if not (0 not in shape and 0 not in keys):
        _check(False, "flux::window_attention: tensor dimensions must be non-empty")
    if not (shape[0] == keys[0]):
        _check(False, "flux::window_attention: batch sizes must match")
    if not (shape[3] == keys[3] and shape[3] <= _MAX_DIM):
        _check(False, "flux::window_attention: head dimensions must match and be at most 256")
    if not (shape[1] % keys[1] == 0):
        _check(False, "flux::window_attention: query heads must be divisible by KV heads")
    if not (keys[2] <= _MAX_KEYS):
        _check(False, "flux::window_attention: more than 16777216 keys")
    if not (key.device == device and value.device == device):
        _check(False, "flux::window_attention: tensor devices must match")
    if not (key.stride(3) == 1 and value.stride(3) == 1 or keys[3] == 1):
        _check(False, "flux::window_attention: key and value must have unit stride along the head dimension")
    if lengths is not None:
        _check_list(lengths, torch.int64, device,
                    "flux::window_attention: lengths must be a contiguous int64 vector on the query device",
                    shape[0], "flux::window_attention: lengths must have one entry per sequence")
    if starts is not None:
        _check_list(starts, torch.int64, device,
                    "flux::window_attention: starts must be a contiguous int64 vector on the query device",
                    shape[0], "flux::window_attention: starts must have one entry per sequence")
    if not (0 <= window <= _MAX_KEYS and 0 <= sinks <= _MAX_KEYS):
        _check(False, "flux::window_attention: window and sinks must be within [0, 16777216]")
    if not (_finite_fp32(scale)):
        _check(False, "flux::window_attention: scale must be a finite FP32 value")
    if torch.is_grad_enabled():
        _grad_free("flux::window_attention", query, key, value)


def _window_cuda(query, key, value, scale, window, sinks=0, lengths=None, starts=None):
    _validate_window(query, key, value, scale, window, sinks, lengths, starts)
    _check(query.is_cuda, "flux::window_attention: CUDA dispatch requires CUDA tensors")
    batch, heads, queries, dim = query.shape
    kv_heads, keys = key.shape[1], key.shape[2]
    output = query.new_empty(query.shape)
    needed, workspace = 0, None
    if queries == 1:
        needed = _size_from("flux_window_attention_workspace_bytes", batch, heads, kv_heads, 1, dim, keys, window, sinks)
        workspace = query.new_empty(needed // 4, dtype=torch.float32)
    _launch("flux_window_attention", query.device, _TYPES[query.dtype], query.data_ptr(), key.data_ptr(), value.data_ptr(),
            _address(lengths), _address(starts), output.data_ptr(), _address(workspace), needed, scale, batch, heads,
            kv_heads, queries, keys, dim, window, sinks, _four(*query.stride()), _four(*key.stride()),
            _four(*value.stride()))
    return output


# ---------------------------------------------------------------------------
# Pages.

def _written_once(tensor) -> bool:
    """No two elements of a tensor that is written share memory: each dimension steps over all smaller ones."""
    if tensor.is_contiguous():
        return True
    reach = 0
    for step, size in sorted((step, size) for step, size in zip(tensor.stride(), tensor.shape) if size > 1):
        if step <= reach:
            return False
        reach += step * (size - 1)
    return True


def _pools_apart(key_pages, value_pages) -> bool:
    """No element of one lies in the other: one ends before the other starts, or, where they are interleaved, every step is
    below a period or a multiple of it, and the parts below it lie apart in it."""
    size = key_pages.element_size()
    between = value_pages.data_ptr() - key_pages.data_ptr()
    if key_pages.is_contiguous() and value_pages.is_contiguous():
        return abs(between) >= key_pages.numel() * size
    key, value = ([(step, count) for step, count in zip(pages.stride(), pages.shape) if count > 1]
                  for pages in (key_pages, value_pages))

    def reach(steps, below):
        return sum(step * (count - 1) for step, count in steps if step < below)

    if between >= (reach(key, math.inf) + 1) * size or -between >= (reach(value, math.inf) + 1) * size:
        return True
    if between % size:
        return False
    for period, _ in key:
        offset = between // size % period
        if (reach(key, period) < offset and offset + reach(value, period) < period and
                not any(step % period for step, _ in key + value if step >= period)):
            return True
    return False


def _validate_pool_memory(op, key_pages, value_pages) -> None:
    """For CPU tensors; the C entries look themselves."""
    _check(_pools_apart(key_pages, value_pages), f"{op}: key and value pages must not overlap")


def _validate_pools(op, key_pages, value_pages, ranks=(4, 5)) -> None:
    shape, dtype, key_stride, value_stride = key_pages.shape, key_pages.dtype, key_pages.stride(), value_pages.stride()
    if len(shape) not in ranks or len(value_stride) != len(shape):
        _check(False, f"{op}: key_pages and value_pages must be [pages, kv_heads, page_size, head_dim]" +
               (", or that behind a layer dimension" if 5 in ranks else ""))
    if dtype not in _TYPES or value_pages.dtype is not dtype:
        _check(False, f"{op}: pages must share dtype float32, float16 or bfloat16")
    if shape != value_pages.shape:
        _check(False, f"{op}: key and value page shapes must match")
    if 0 in shape:
        _check(False, f"{op}: pages must be non-empty")
    if key_pages.device != value_pages.device:
        _check(False, f"{op}: tensor devices must match")
    if (key_stride[-1] != 1 or value_stride[-1] != 1) and shape[-1] != 1:
        _check(False, f"{op}: pages must have unit stride along the head dimension")
    if not _written_once(key_pages):
        _check(False, f"{op}: key_pages must not overlap itself")
    if not _written_once(value_pages):
        _check(False, f"{op}: value_pages must not overlap itself")
    if key_pages.is_set_to(value_pages):
        _check(False, f"{op}: key_pages and value_pages must not be the same memory")
    if torch.is_grad_enabled():
        _grad_free(op, key_pages, value_pages)


def _validate_table(op, page_table) -> None:
    shape = page_table.shape
    if len(shape) != 2 or page_table.dtype is not torch.int32 or 0 in shape:
        _check(False, f"{op}: page_table must be int32 [slots, columns]")
    if page_table.stride(1) != 1 and shape[1] != 1:
        _check(False, f"{op}: page_table rows must be contiguous")


def _validate_books(op, page_table, lengths, refcounts) -> None:
    _validate_table(op, page_table)
    slots, columns = page_table.shape
    if page_table.stride(0) < columns and slots != 1:
        _check(False, f"{op}: page_table rows must not overlap")
    device = page_table.device
    if lengths is not None:
        if (lengths.dim() != 1 or lengths.dtype is not torch.int64 or lengths.device != device or
                not lengths.is_contiguous()):
            _check(False, f"{op}: lengths must be a contiguous int64 vector on the page_table device")
        if lengths.shape[0] != slots:
            _check(False, f"{op}: lengths must have one entry per page_table row")
    if (refcounts.dim() != 1 or refcounts.dtype is not torch.int32 or refcounts.device != device or
            not refcounts.is_contiguous()):
        _check(False, f"{op}: refcounts must be a contiguous int32 vector on the page_table device")
    if refcounts.shape[0] == 0:
        _check(False, f"{op}: refcounts must have one entry per page")


def _validate_requests(op, name, requests, like) -> None:
    if (requests.dim() != 1 or requests.dtype is not torch.int64 or requests.device != like.device or
            not requests.is_contiguous()):
        _check(False, f"{op}: {name} must be a contiguous int64 vector on the cache's device")


def _pool(key_pages, value_pages) -> bytes:
    layers, *shape = key_pages.shape if key_pages.dim() == 5 else (1, *key_pages.shape)
    key_strides, value_strides = key_pages.stride(), value_pages.stride()
    if len(key_strides) == 4:
        key_strides, value_strides = (0, *key_strides), (0, *value_strides)
    return _page_pool(key_pages.data_ptr(), value_pages.data_ptr(), layers, *shape, *key_strides[:4], *value_strides[:4],
                      _TYPES[key_pages.dtype])


def _books(page_table, lengths, refcounts, page_size) -> bytes:
    return _page_books(page_table.data_ptr(), page_table.stride(0), *page_table.shape,
                       0 if lengths is None else lengths.data_ptr(), refcounts.data_ptr(), refcounts.shape[0], page_size)


def _page_size_of(key_pages) -> int:
    return key_pages.shape[-2]


def _validate_reserve(page_table, lengths, refcounts, page_size, slots, counts=None) -> None:
    op = "flux::paged_cache_reserve"
    _validate_books(op, page_table, lengths, refcounts)
    if not (page_size > 0 and page_table.shape[1] * page_size <= _MAX_KEYS):
        _check(False, f"{op}: page_size must be positive and a page_table row hold at most 16777216 positions")
    _validate_requests(op, "slots", slots, page_table)
    if counts is not None:
        _validate_requests(op, "counts", counts, page_table)
        _check(counts.shape == slots.shape, f"{op}: counts must have one entry per slot")


def _reserve_cuda(page_table, lengths, refcounts, page_size, slots, counts=None):
    _validate_reserve(page_table, lengths, refcounts, page_size, slots, counts)
    _require_gpu("flux::paged_cache_reserve", page_table)
    requests = slots.shape[0]
    positions = torch.empty_like(slots)
    status = page_table.new_empty(requests)
    if requests == 0:
        return positions, status
    words = _size_from("flux_page_reserve_workspace_words", requests, page_table.shape[0], refcounts.shape[0])
    workspace = page_table.new_empty(words)
    _launch("flux_page_reserve", slots.device, _books(page_table, lengths, refcounts, page_size), slots.data_ptr(),
            _address(counts), requests, positions.data_ptr(), status.data_ptr(), workspace.data_ptr(), words)
    return positions, status


def _validate_write(key, value, key_pages, value_pages, page_table, slots, positions, counts=None) -> None:
    op = "flux::paged_cache_write"
    _validate_pools(op, key_pages, value_pages, (4,))
    _validate_table(op, page_table)
    shape, pages, dtype, device = key.shape, key_pages.shape, key_pages.dtype, key_pages.device
    if not (page_table.device == device):
        _check(False, "flux::paged_cache_write: tensor devices must match")
    if not (page_table.shape[1] * pages[2] <= _MAX_KEYS):
        _check(False, "flux::paged_cache_write: page_table holds more than 16777216 positions a row")
    if not (len(shape) == 4 and value.shape == shape):
        _check(False, "flux::paged_cache_write: key and value must be rank four and of one shape")
    if not (key.dtype is dtype and value.dtype is dtype and key.device == device and value.device == device):
        _check(False, "flux::paged_cache_write: key and value must have the pages' dtype and device")
    if not (shape[1] == pages[1] and shape[3] == pages[3]):
        _check(False, "flux::paged_cache_write: key heads and head dimension must be the pages'")
    if not (key.stride(3) == 1 and value.stride(3) == 1 or shape[3] == 1):
        _check(False, "flux::paged_cache_write: key and value must have unit stride along the head dimension")
    requests = shape[0]
    _check_list(slots, torch.int64, device,
                "flux::paged_cache_write: slots must be a contiguous int64 vector on the cache's device",
                requests, "flux::paged_cache_write: slots must have one entry per request")
    _check_list(positions, torch.int64, device,
                "flux::paged_cache_write: positions must be a contiguous int64 vector on the cache's device",
                requests, "flux::paged_cache_write: positions must have one entry per request")
    if counts is not None:
        _check_list(counts, torch.int64, device,
                    "flux::paged_cache_write: counts must be a contiguous int64 vector on the cache's device",
                    requests, "flux::paged_cache_write: counts must have one entry per request")
    if not (requests <= 65535):
        _check(False, "flux::paged_cache_write: more than 65535 requests")
    if torch.is_grad_enabled():
        _grad_free(op, key, value)


def _validate_write_memory(key, value, key_pages, value_pages, page_table, slots, positions, counts=None) -> None:
    _validate_write(key, value, key_pages, value_pages, page_table, slots, positions, counts)
    stores = key_pages.untyped_storage().data_ptr(), value_pages.untyped_storage().data_ptr()
    _check(key.untyped_storage().data_ptr() not in stores and value.untyped_storage().data_ptr() not in stores,
           "flux::paged_cache_write: the pages must not alias key or value")


def _validate_write_pools(key, value, key_pages, value_pages, page_table, slots, positions, counts=None) -> None:
    _validate_write_memory(key, value, key_pages, value_pages, page_table, slots, positions, counts)
    _validate_pool_memory("flux::paged_cache_write", key_pages, value_pages)


def _write_cuda(key, value, key_pages, value_pages, page_table, slots, positions, counts=None):
    _validate_write_memory(key, value, key_pages, value_pages, page_table, slots, positions, counts)
    _require_gpu("flux::paged_cache_write", key_pages)
    if key.shape[0] == 0 or key.shape[2] == 0:
        return
    _launch("flux_page_write", key_pages.device, _pool(key_pages, value_pages), key.data_ptr(), value.data_ptr(),
            _four(*key.stride()), _four(*value.stride()), key.shape[0], key.shape[2], page_table.data_ptr(),
            page_table.stride(0), *page_table.shape, slots.data_ptr(), positions.data_ptr(), _address(counts))


def _validate_copy(key_pages, value_pages, source, target) -> None:
    op = "flux::paged_cache_copy"
    _validate_pools(op, key_pages, value_pages)
    _validate_requests(op, "source", source, key_pages)
    _validate_requests(op, "target", target, key_pages)
    if not (source.shape == target.shape):
        _check(False, f"{op}: source and target must have one length")


def _validate_copy_pools(key_pages, value_pages, source, target) -> None:
    _validate_copy(key_pages, value_pages, source, target)
    _validate_pool_memory("flux::paged_cache_copy", key_pages, value_pages)


def _copy_cuda(key_pages, value_pages, source, target):
    _validate_copy(key_pages, value_pages, source, target)
    _require_gpu("flux::paged_cache_copy", key_pages)
    status = source.new_empty(source.shape[0], dtype=torch.int32)
    if source.shape[0]:
        _launch("flux_page_copy", source.device, _pool(key_pages, value_pages), source.data_ptr(), target.data_ptr(),
                source.shape[0], status.data_ptr())
    return status


def _validate_free(page_table, lengths, refcounts, slots) -> None:
    op = "flux::paged_cache_free"
    _validate_books(op, page_table, lengths, refcounts)
    _validate_requests(op, "slots", slots, page_table)


def _free_cuda(page_table, lengths, refcounts, slots):
    _validate_free(page_table, lengths, refcounts, slots)
    _require_gpu("flux::paged_cache_free", page_table)
    status = page_table.new_empty(slots.shape[0])
    if slots.shape[0]:
        _launch("flux_page_free", slots.device, _books(page_table, lengths, refcounts, 1), slots.data_ptr(),
                slots.shape[0], status.data_ptr())
    return status


def _validate_fork(key_pages, value_pages, page_table, lengths, refcounts, parents, children) -> None:
    op = "flux::paged_cache_fork"
    _validate_pools(op, key_pages, value_pages)
    _validate_books(op, page_table, lengths, refcounts)
    if not (page_table.device == key_pages.device):
        _check(False, f"{op}: tensor devices must match")
    if not (refcounts.shape[0] == key_pages.shape[-4]):
        _check(False, f"{op}: refcounts must have one entry per page")
    if not (page_table.shape[1] * key_pages.shape[-2] <= _MAX_KEYS):
        _check(False, f"{op}: page_table holds more than 16777216 positions a row")
    _validate_requests(op, "parents", parents, key_pages)
    _validate_requests(op, "children", children, key_pages)
    if not (parents.shape == children.shape):
        _check(False, f"{op}: parents and children must have one length")


def _validate_fork_pools(key_pages, value_pages, page_table, lengths, refcounts, parents, children) -> None:
    _validate_fork(key_pages, value_pages, page_table, lengths, refcounts, parents, children)
    _validate_pool_memory("flux::paged_cache_fork", key_pages, value_pages)


def _fork_cuda(key_pages, value_pages, page_table, lengths, refcounts, parents, children):
    _validate_fork(key_pages, value_pages, page_table, lengths, refcounts, parents, children)
    _require_gpu("flux::paged_cache_fork", key_pages)
    requests = parents.shape[0]
    status = page_table.new_empty(requests)
    if requests == 0:
        return status
    words = _size_from("flux_page_fork_workspace_words", requests, page_table.shape[0], refcounts.shape[0])
    workspace = page_table.new_empty(words)
    _launch("flux_page_fork", parents.device, _pool(key_pages, value_pages),
            _books(page_table, lengths, refcounts, _page_size_of(key_pages)), parents.data_ptr(), children.data_ptr(),
            requests, status.data_ptr(), workspace.data_ptr(), words)
    return status


def _validate_compact(key_pages, value_pages, page_table, refcounts) -> None:
    op = "flux::paged_cache_compact"
    _validate_pools(op, key_pages, value_pages)
    _validate_books(op, page_table, None, refcounts)
    if not (page_table.device == key_pages.device):
        _check(False, f"{op}: tensor devices must match")
    if not (refcounts.shape[0] == key_pages.shape[-4]):
        _check(False, f"{op}: refcounts must have one entry per page")


def _validate_compact_pools(key_pages, value_pages, page_table, refcounts) -> None:
    _validate_compact(key_pages, value_pages, page_table, refcounts)
    _validate_pool_memory("flux::paged_cache_compact", key_pages, value_pages)


def _compact_cuda(key_pages, value_pages, page_table, refcounts):
    _validate_compact(key_pages, value_pages, page_table, refcounts)
    _require_gpu("flux::paged_cache_compact", key_pages)
    pages = refcounts.shape[0]
    page_map = refcounts.new_empty(pages)
    used = refcounts.new_empty((), dtype=torch.int64)
    words = _size_from("flux_page_compact_workspace_words", pages)
    workspace = refcounts.new_empty(words)
    _launch("flux_page_compact", refcounts.device, _pool(key_pages, value_pages),
            _books(page_table, None, refcounts, _page_size_of(key_pages)), page_map.data_ptr(), used.data_ptr(),
            workspace.data_ptr(), words)
    return page_map, used


# ---------------------------------------------------------------------------
# logits_process

def _validate_penalty(name, penalty, device, rows, history) -> None:
    if (penalty.dim() != 1 or penalty.dtype is not torch.float32 or penalty.device != device or
            not penalty.is_contiguous()):
        _check(False, f"flux::logits_process: {name} must be a contiguous float32 vector on the logits device")
    if penalty.shape[0] != rows:
        _check(False, f"flux::logits_process: {name} must have one entry per row")
    if history is None:
        _check(False, f"flux::logits_process: {name} needs a history")


def _validate_logits(logits, history=None, history_lengths=None, repetition=None, frequency=None, presence=None,
                     bias=None, allowed=None) -> None:
    shape, device = logits.shape, logits.device
    if not (len(shape) == 2 and shape[0] > 0 and 0 < shape[1] <= _MAX_VOCAB):
        _check(False, "flux::logits_process: logits must be [rows, vocab], non-empty, vocab at most 16777216")
    if not (logits.dtype in _TYPES):
        _check(False, "flux::logits_process: logits must have dtype float32, float16 or bfloat16")
    rows, vocab = shape
    if not (logits.stride(1) == 1 or vocab == 1):
        _check(False, "flux::logits_process: logits rows must be contiguous")
    if history is not None:
        width = history.shape
        _check(len(width) == 2 and width[0] == rows and history.dtype is torch.int64,
               "flux::logits_process: history must be int64 [rows, width]")
        _check(history.stride(1) == 1 or width[1] <= 1, "flux::logits_process: history rows must be contiguous")
        _check(history.device == device, "flux::logits_process: tensor devices must match")
    if not (history is not None or history_lengths is None):
        _check(False, "flux::logits_process: history_lengths needs a history")
    if history_lengths is not None:
        _check_list(history_lengths, torch.int64, device,
                    "flux::logits_process: history_lengths must be a contiguous int64 vector on the logits device",
                    rows, "flux::logits_process: history_lengths must have one entry per row")
    if repetition is not None:
        _validate_penalty("repetition", repetition, device, rows, history)
    if frequency is not None:
        _validate_penalty("frequency", frequency, device, rows, history)
    if presence is not None:
        _validate_penalty("presence", presence, device, rows, history)
    if bias is not None:
        width = bias.shape
        _check(len(width) == 2 and width[0] in (1, rows) and width[1] == vocab and bias.dtype is torch.float32 and
               bias.device == device, "flux::logits_process: bias must be float32 [1 or rows, vocab] on the logits device")
        _check(bias.stride(1) == 1 or vocab == 1, "flux::logits_process: bias rows must be contiguous")
    if allowed is not None:
        width = allowed.shape
        _check(len(width) == 2 and width[0] in (1, rows) and width[1] == (vocab + 31) // 32 and
               allowed.dtype is torch.int32 and allowed.device == device,
               "flux::logits_process: allowed must be int32 [1 or rows, ceil(vocab / 32)] on the logits device")
        _check(allowed.stride(1) == 1 or width[1] == 1, "flux::logits_process: allowed rows must be contiguous")
    if torch.is_grad_enabled():
        _grad_free("flux::logits_process", logits, bias, repetition, frequency, presence)


def _row_stride(tensor) -> int:
    return 0 if tensor is None or tensor.shape[0] == 1 else tensor.stride(0)


def _logits_cuda(logits, history=None, history_lengths=None, repetition=None, frequency=None, presence=None, bias=None,
                 allowed=None):
    _validate_logits(logits, history, history_lengths, repetition, frequency, presence, bias, allowed)
    _require_gpu("flux::logits_process", logits)
    rows, vocab = logits.shape
    processed = logits.new_empty((rows, vocab))
    tokens = logits.new_empty(rows, dtype=torch.int64)
    needed = _size_from("flux_logits_process_workspace_bytes", rows, vocab)
    workspace = tokens.new_empty(needed // 8) if needed else None
    _launch("flux_logits_process", logits.device, _TYPES[logits.dtype], logits.data_ptr(), logits.stride(0),
            processed.data_ptr(), tokens.data_ptr(), rows, vocab, _address(history),
            0 if history is None else history.shape[1], 0 if history is None else history.stride(0),
            _address(history_lengths), _address(repetition), _address(frequency), _address(presence), _address(bias),
            _row_stride(bias), _address(allowed), _row_stride(allowed), _address(workspace), needed)
    return processed, tokens


# ---------------------------------------------------------------------------
# Dispatcher registration.

_KERNELS = {
    "paged_decode_attention": (_paged_cuda, _validate_paged),
    "paged_decode_attention_out": (_paged_out_cuda, _validate_paged_out_memory),
    "window_attention": (_window_cuda, _validate_window),
    "paged_cache_reserve": (_reserve_cuda, _validate_reserve),
    "paged_cache_write": (_write_cuda, _validate_write_pools),
    "paged_cache_copy": (_copy_cuda, _validate_copy_pools),
    "paged_cache_fork": (_fork_cuda, _validate_fork_pools),
    "paged_cache_free": (_free_cuda, _validate_free),
    "paged_cache_compact": (_compact_cuda, _validate_compact_pools),
    "logits_process": (_logits_cuda, _validate_logits),
}

for _name, (_cuda, _validate) in _KERNELS.items():
    _LIBRARY.impl(_name, _cuda, "CUDA")
    _LIBRARY.impl(_name, _cpu_kernel(_name, _validate), "CPU")


@torch.library.register_fake("flux::paged_decode_attention")
def _paged_fake(query, key_pages, value_pages, page_table, lengths, scale, window=0, sinks=0, slots=None):
    _validate_paged(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots)
    return query.new_empty(query.shape)


@torch.library.register_fake("flux::paged_decode_attention_out")
def _paged_out_fake(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots, output, workspace):
    _validate_paged_out(query, key_pages, value_pages, page_table, lengths, scale, window, sinks, slots, output,
                        workspace)
    return output


@torch.library.register_fake("flux::window_attention")
def _window_fake(query, key, value, scale, window, sinks=0, lengths=None, starts=None):
    _validate_window(query, key, value, scale, window, sinks, lengths, starts)
    return query.new_empty(query.shape)


@torch.library.register_fake("flux::paged_cache_reserve")
def _reserve_fake(page_table, lengths, refcounts, page_size, slots, counts=None):
    _validate_reserve(page_table, lengths, refcounts, page_size, slots, counts)
    return slots.new_empty(slots.shape), slots.new_empty(slots.shape, dtype=torch.int32)


@torch.library.register_fake("flux::paged_cache_write")
def _write_fake(key, value, key_pages, value_pages, page_table, slots, positions, counts=None):
    _validate_write(key, value, key_pages, value_pages, page_table, slots, positions, counts)


@torch.library.register_fake("flux::paged_cache_copy")
def _copy_fake(key_pages, value_pages, source, target):
    _validate_copy(key_pages, value_pages, source, target)
    return source.new_empty(source.shape, dtype=torch.int32)


@torch.library.register_fake("flux::paged_cache_fork")
def _fork_fake(key_pages, value_pages, page_table, lengths, refcounts, parents, children):
    _validate_fork(key_pages, value_pages, page_table, lengths, refcounts, parents, children)
    return parents.new_empty(parents.shape, dtype=torch.int32)


@torch.library.register_fake("flux::paged_cache_free")
def _free_fake(page_table, lengths, refcounts, slots):
    _validate_free(page_table, lengths, refcounts, slots)
    return slots.new_empty(slots.shape, dtype=torch.int32)


@torch.library.register_fake("flux::paged_cache_compact")
def _compact_fake(key_pages, value_pages, page_table, refcounts):
    _validate_compact(key_pages, value_pages, page_table, refcounts)
    return refcounts.new_empty(refcounts.shape), refcounts.new_empty((), dtype=torch.int64)


@torch.library.register_fake("flux::logits_process")
def _logits_fake(logits, history=None, history_lengths=None, repetition=None, frequency=None, presence=None, bias=None,
                 allowed=None):
    _validate_logits(logits, history, history_lengths, repetition, frequency, presence, bias, allowed)
    return logits.new_empty(logits.shape), logits.new_empty((logits.shape[0],), dtype=torch.int64)


# ---------------------------------------------------------------------------
# Python entry points.  They call the overloads themselves: looking one up by its packet costs 2 us a call.

class _Overloads:
    __slots__ = SERVING_OPERATOR_NAMES

    def __init__(self) -> None:
        for name in SERVING_OPERATOR_NAMES:
            setattr(self, name, getattr(torch.ops.flux, name).default)


_OPS = _Overloads()


def native_paged_decode_attention_is_available() -> bool:
    return _availability("paged_decode_attention", "paged_decode_attention_out")


def native_window_attention_is_available() -> bool:
    return _availability("window_attention")


def native_paged_cache_is_available() -> bool:
    return _availability(*(name for name in SERVING_SCHEMAS if name.startswith("paged_cache_")))


def native_logits_process_is_available() -> bool:
    return _availability("logits_process")


def paged_decode_attention_native(query: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                                  page_table: torch.Tensor, lengths: torch.Tensor, scale: float, window: int = 0,
                                  sinks: int = 0, slots: torch.Tensor | None = None) -> torch.Tensor:
    """One-token GQA attention of a batch over its cache pages; the new token's rows are already in them.

    ``query`` [B, Hq, 1, D], pages [P, Hkv, page_size, D] (any strides, D contiguous); sequence b uses row ``slots[b]``
    (b without slots) of ``page_table`` and ``lengths``.  ``window`` > 0 leaves the last ``window`` keys and the first
    ``sinks`` visible.  Keys on an entry outside [0, P) are left out; a sequence that sees nothing gives zeros.
    """
    _ready("paged decode attention")
    return _OPS.paged_decode_attention(query, key_pages, value_pages, page_table, lengths, scale, window,
                                                 sinks, slots)


def paged_decode_attention_native_out(query: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                                      page_table: torch.Tensor, lengths: torch.Tensor, scale: float, window: int,
                                      sinks: int, slots: torch.Tensor | None, output: torch.Tensor,
                                      workspace: torch.Tensor) -> torch.Tensor:
    """The same into stable buffers (float32 workspace of at least ``paged_decode_workspace_bytes``); returns ``output``.

    Calls that may overlap need workspaces of their own.
    """
    _ready("paged decode attention out variant")
    return _OPS.paged_decode_attention_out(query, key_pages, value_pages, page_table, lengths, scale, window,
                                                     sinks, slots, output, workspace)


def window_attention_native(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, scale: float, window: int,
                            sinks: int = 0, lengths: torch.Tensor | None = None,
                            starts: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA attention with a sliding window and sinks: prompts, chunks of them, single tokens.

    ``query`` [B, Hq, S, D] over ``key``, ``value`` [B, Hkv, L, D].  Query i of sequence b is at position
    ``starts[b] + i`` (default ``lengths[b] - S + i``, lengths by default L) and sees the keys j up to its own with
    ``j > position - window`` or ``j < sinks``; window 0 leaves all of them visible.  Rows whose position is not a
    key's give zeros: a padded batch of prompts passes ``starts`` of zeros and its lengths.
    """
    _ready("window attention")
    return _OPS.window_attention(query, key, value, scale, window, sinks, lengths, starts)


def paged_cache_reserve_native(page_table: torch.Tensor, lengths: torch.Tensor, refcounts: torch.Tensor, page_size: int,
                               slots: torch.Tensor, counts: torch.Tensor | None = None
                               ) -> tuple[torch.Tensor, torch.Tensor]:
    """Pages for the next ``counts`` (default one) tokens of ``slots``; returns (first positions, status).

    Columns without a page get the lowest free ones, in the order of the requests, and ``lengths`` grow.  A request that
    cannot be served changes nothing and has position -1.
    """
    _ready("paged cache")
    return _OPS.paged_cache_reserve(page_table, lengths, refcounts, page_size, slots, counts)


def paged_cache_write_native(key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                             page_table: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
                             counts: torch.Tensor | None = None) -> None:
    """Rows of new tokens ``key``, ``value`` [N, Hkv, S, D] of one layer to ``positions`` (and on) of ``slots``.

    Only the first ``counts[i]`` tokens of request i are written.  Negative positions (refused reservations) and rows on
    no page are skipped; two requests must not name the same rows.
    """
    _ready("paged cache")
    _OPS.paged_cache_write(key, value, key_pages, value_pages, page_table, slots, positions, counts)


def paged_cache_copy_native(key_pages: torch.Tensor, value_pages: torch.Tensor, source: torch.Tensor,
                            target: torch.Tensor) -> torch.Tensor:
    """Pages ``source`` to pages ``target`` in all layers; returns the status of each pair."""
    _ready("paged cache")
    return _OPS.paged_cache_copy(key_pages, value_pages, source, target)


def paged_cache_fork_native(key_pages: torch.Tensor, value_pages: torch.Tensor, page_table: torch.Tensor,
                            lengths: torch.Tensor, refcounts: torch.Tensor, parents: torch.Tensor,
                            children: torch.Tensor) -> torch.Tensor:
    """The empty slots ``children`` become branches of ``parents``; returns the status of each.

    Full pages are shared, the rows of a partial last page are copied to a new page, so both may write on.
    """
    _ready("paged cache")
    return _OPS.paged_cache_fork(key_pages, value_pages, page_table, lengths, refcounts, parents, children)


def paged_cache_free_native(page_table: torch.Tensor, lengths: torch.Tensor, refcounts: torch.Tensor,
                            slots: torch.Tensor) -> torch.Tensor:
    """Empties ``slots``: their pages lose a holder each, and those without one are free; returns the status of each."""
    _ready("paged cache")
    return _OPS.paged_cache_free(page_table, lengths, refcounts, slots)


def paged_cache_compact_native(key_pages: torch.Tensor, value_pages: torch.Tensor, page_table: torch.Tensor,
                               refcounts: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Moves the pages in use to the front of the pool; returns (page_map int32 [P], pages in use).

    ``page_table`` and ``refcounts`` follow; ``page_map`` gives each page's new place (-1: free) for what else names one.
    """
    _ready("paged cache")
    return _OPS.paged_cache_compact(key_pages, value_pages, page_table, refcounts)


def logits_process_native(logits: torch.Tensor, history: torch.Tensor | None = None,
                          history_lengths: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                          frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                          bias: torch.Tensor | None = None, allowed: torch.Tensor | None = None
                          ) -> tuple[torch.Tensor, torch.Tensor]:
    """Penalties, bias and grammar mask on ``logits`` [rows, vocab]; returns (processed logits, greedy tokens).

    A token that occurs c > 0 times in the first ``history_lengths`` ids of the row's ``history`` becomes ``x /
    repetition`` (``x * repetition`` when not positive), minus ``frequency * c``, minus ``presence``; then ``bias`` is
    added and tokens whose bit of ``allowed`` (bit v % 32 of word v // 32) is clear become -inf.  The greedy token is the
    lowest index of the largest processed logit (NaN above all numbers).
    """
    _ready("logits process")
    return _OPS.logits_process(logits, history, history_lengths, repetition, frequency, presence, bias, allowed)

