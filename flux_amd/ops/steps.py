"""``torch.ops.flux.*`` for served steps in which chunks of prompts and single tokens run together.

The step's tokens lie packed, one request after the other: ``[tokens, ...]`` with ``offsets`` int64 ``[requests + 1]``.
``paged_step_layout`` derives them, each token's position and its row of the page pool from the requests that
``paged_cache_reserve`` served; ``paged_cache_write_rows`` and ``paged_chunk_attention`` take them in every layer, and
``logits_sample`` ends the step.  Cache, books and manner are those of ``flux_amd.ops.serving``.
"""

from __future__ import annotations

import struct

import torch

from flux_amd.ops.native import _LIBRARY, _availability, _check, _cpu_kernel, _finite_fp32, _grad_free, _require_gpu
from flux_amd.ops.serving import (_MAX_DIM, _MAX_KEYS, _MAX_VOCAB, _TYPES, _address, _check_list, _launch, _pool, _ready,
                                  _size_from, _validate_pool_memory, _validate_pools, _validate_table)

STEP_SCHEMAS = {
    "paged_step_layout": ("paged_step_layout(Tensor page_table, Tensor slots, Tensor positions, Tensor? counts, "
                          "int page_size, int tokens) -> (Tensor offsets, Tensor token_requests, Tensor token_positions, "
                          "Tensor token_rows)"),
    "paged_cache_write_rows": ("paged_cache_write_rows(Tensor key, Tensor value, Tensor(a!) key_pages, "
                               "Tensor(b!) value_pages, Tensor rows) -> ()"),
    "paged_chunk_attention": ("paged_chunk_attention(Tensor query, Tensor key_pages, Tensor value_pages, Tensor page_table, "
                              "Tensor lengths, Tensor offsets, float scale, int window=0, int sinks=0, "
                              "Tensor? slots=None, Tensor? positions=None) -> Tensor"),
    "logits_sample": ("logits_sample(Tensor logits, Tensor uniforms, Tensor? temperature=None, Tensor? top_k=None, "
                      "Tensor? top_p=None, Tensor? min_p=None) -> (Tensor tokens, Tensor probabilities)"),
}

STEP_OPERATOR_NAMES = tuple(STEP_SCHEMAS)

for _schema in STEP_SCHEMAS.values():
    _LIBRARY.define(_schema)

_MAX_REQUESTS = 65535
_two, _three = struct.Struct("2q").pack, struct.Struct("3q").pack


# ---------------------------------------------------------------------------
# paged_step_layout

def _validate_layout(page_table, slots, positions, counts, page_size, tokens) -> None:
    _validate_table("flux::paged_step_layout", page_table)
    device = page_table.device
    if not (page_size > 0 and page_table.shape[1] * page_size <= _MAX_KEYS):
        _check(False, "flux::paged_step_layout: page_size must be positive and a page_table row hold at most 16777216 "
                      "positions")
    if not (0 <= tokens <= _MAX_KEYS):
        _check(False, "flux::paged_step_layout: tokens must be within [0, 16777216]")
    _check_list(slots, torch.int64, device,
                "flux::paged_step_layout: slots must be a contiguous int64 vector on the page_table device")
    requests = slots.shape[0]
    if not (requests <= _MAX_REQUESTS):
        _check(False, "flux::paged_step_layout: more than 65535 requests")
    _check_list(positions, torch.int64, device,
                "flux::paged_step_layout: positions must be a contiguous int64 vector on the page_table device",
                requests, "flux::paged_step_layout: positions must have one entry per request")
    if counts is not None:
        _check_list(counts, torch.int64, device,
                    "flux::paged_step_layout: counts must be a contiguous int64 vector on the page_table device",
                    requests, "flux::paged_step_layout: counts must have one entry per request")


def _layout_cuda(page_table, slots, positions, counts, page_size, tokens):
    _validate_layout(page_table, slots, positions, counts, page_size, tokens)
    _require_gpu("flux::paged_step_layout", page_table)
    requests = slots.shape[0]
    if requests == 0 or tokens == 0:
        return slots.new_zeros(requests + 1), *(slots.new_full((tokens,), -1) for _ in range(3))
    offsets = slots.new_empty(requests + 1)
    of, at, rows = (slots.new_empty(tokens) for _ in range(3))
    _launch("flux_step_layout", slots.device, page_table.data_ptr(), page_table.stride(0), *page_table.shape, page_size,
            slots.data_ptr(), positions.data_ptr(), _address(counts), requests, tokens, offsets.data_ptr(), of.data_ptr(),
            at.data_ptr(), rows.data_ptr())
    return offsets, of, at, rows


# ---------------------------------------------------------------------------
# paged_cache_write_rows

def _validate_rows(key, value, key_pages, value_pages, rows) -> None:
    op = "flux::paged_cache_write_rows"
    _validate_pools(op, key_pages, value_pages, (4,))
    shape, pages, dtype, device = key.shape, key_pages.shape, key_pages.dtype, key_pages.device
    if not (len(shape) == 3 and value.shape == shape):
        _check(False, "flux::paged_cache_write_rows: key and value must be [tokens, kv_heads, head_dim] and of one shape")
    if not (key.dtype is dtype and value.dtype is dtype and key.device == device and value.device == device):
        _check(False, "flux::paged_cache_write_rows: key and value must have the pages' dtype and device")
    if not (shape[1] == pages[1] and shape[2] == pages[3]):
        _check(False, "flux::paged_cache_write_rows: key heads and head dimension must be the pages'")
    if not (key.stride(2) == 1 and value.stride(2) == 1 or shape[2] == 1):
        _check(False, "flux::paged_cache_write_rows: key and value must have unit stride along the head dimension")
    if not (shape[0] <= _MAX_KEYS):
        _check(False, "flux::paged_cache_write_rows: more than 16777216 tokens")
    if not (pages[0] <= 1 << 28 and pages[2] <= _MAX_KEYS and max(pages[1], pages[3]) <= 1 << 20 and pages[1] * pages[3] <= 1 << 24 and
            pages[1] * pages[2] * pages[3] <= 1 << 28):
        _check(False, "flux::paged_cache_write_rows: more than 268435456 pages or elements a page, 16777216 rows a page or elements "
                      "a token, or 1048576 heads or dims")
    _check_list(rows, torch.int64, device,
                "flux::paged_cache_write_rows: rows must be a contiguous int64 vector on the cache's device",
                shape[0], "flux::paged_cache_write_rows: rows must have one entry per token")
    if torch.is_grad_enabled():
        _grad_free(op, key, value)


def _validate_rows_memory(key, value, key_pages, value_pages, rows) -> None:
    _validate_rows(key, value, key_pages, value_pages, rows)
    stores = key_pages.untyped_storage().data_ptr(), value_pages.untyped_storage().data_ptr()
    for tensor in (key, value, rows):
        if tensor.untyped_storage().data_ptr() in stores:
            _check(False, "flux::paged_cache_write_rows: the pages must not alias key, value or rows")


def _validate_rows_pools(key, value, key_pages, value_pages, rows) -> None:
    _validate_rows_memory(key, value, key_pages, value_pages, rows)
    _validate_pool_memory("flux::paged_cache_write_rows", key_pages, value_pages)


def _rows_cuda(key, value, key_pages, value_pages, rows):
    _validate_rows_memory(key, value, key_pages, value_pages, rows)
    _require_gpu("flux::paged_cache_write_rows", key_pages)
    if key.shape[0] == 0:
        return
    _launch("flux_page_write_rows", key_pages.device, _pool(key_pages, value_pages), key.data_ptr(), value.data_ptr(),
            _two(*key.stride()[:2]), _two(*value.stride()[:2]), key.shape[0], rows.data_ptr())


# ---------------------------------------------------------------------------
# paged_chunk_attention

def _workgroups(shape, kv_heads, dtype, requests) -> int:
    """At most, of a call: its tiles, each request's last one partly filled, and what they are cut into."""
    rows = shape[0] * (shape[1] // kv_heads)
    whole = dtype is not torch.float32 or shape[2] <= 64 and rows >= max(64 * requests, 2048)
    tiles = min(rows, rows // (128 if whole else 32 if shape[2] <= 128 else 16) + requests)
    return (tiles + 1024 // kv_heads + 64) * kv_heads


def _validate_chunk(query, key_pages, value_pages, page_table, lengths, offsets, scale, window=0, sinks=0, slots=None,
                    positions=None) -> None:
    shape, pages, table, dtype, device = query.shape, key_pages.shape, page_table.shape, query.dtype, query.device
    if not (len(shape) == 3 and len(pages) == 4 and value_pages.dim() == 4):
        _check(False, "flux::paged_chunk_attention: query must be [tokens, query_heads, head_dim] and pages of rank four")
    if not (dtype in _TYPES and key_pages.dtype is dtype and value_pages.dtype is dtype):
        _check(False, "flux::paged_chunk_attention: query and pages must share dtype float32, float16 or bfloat16")
    if not (pages == value_pages.shape):
        _check(False, "flux::paged_chunk_attention: key and value page shapes must match")
    if not (0 not in shape[1:] and 0 not in pages):
        _check(False, "flux::paged_chunk_attention: heads, head dimension and pages must be non-empty")
    if not (shape[2] == pages[3] and shape[2] <= _MAX_DIM):
        _check(False, "flux::paged_chunk_attention: head dimensions must match and be at most 256")
    if not (shape[1] % pages[1] == 0):
        _check(False, "flux::paged_chunk_attention: query heads must be divisible by KV heads")
    if not (shape[0] <= _MAX_KEYS and shape[0] * (shape[1] // pages[1]) <= 1 << 27):
        _check(False, "flux::paged_chunk_attention: more than 16777216 tokens or 134217728 rows of a KV head")
    if not (shape[1] <= 65535 and pages[0] <= 1 << 28):
        _check(False, "flux::paged_chunk_attention: more than 65535 query heads or 268435456 pages")
    if not (len(table) == 2 and page_table.dtype is torch.int32 and 0 not in table):
        _check(False, "flux::paged_chunk_attention: page_table must be int32 [slots, columns]")
    if not (page_table.stride(1) == 1 or table[1] == 1):
        _check(False, "flux::paged_chunk_attention: page_table rows must be contiguous")
    if not (table[1] * pages[2] <= _MAX_KEYS):
        _check(False, "flux::paged_chunk_attention: page_table holds more than 16777216 positions a row")
    _check_list(lengths, torch.int64, device,
                "flux::paged_chunk_attention: lengths must be a contiguous int64 vector on the query device",
                table[0], "flux::paged_chunk_attention: lengths must have one entry per page_table row")
    _check_list(offsets, torch.int64, device,
                "flux::paged_chunk_attention: offsets must be a contiguous int64 vector on the query device")
    requests = offsets.shape[0] - 1
    if not (0 <= requests <= _MAX_REQUESTS):
        _check(False, "flux::paged_chunk_attention: offsets must have one entry more than the requests, at most 65535")
    # The bound of the smallest tiles first: hardly any call is beyond it.
    if (shape[0] * shape[1] + 16 * ((requests + 64) * pages[1] + 1024) >= 1 << 28 and
            _workgroups(shape, pages[1], dtype, requests) >= 1 << 24):
        _check(False, "flux::paged_chunk_attention: the rows' tiles are 16777216 or more over all KV heads")
    if slots is None:
        _check(table[0] >= requests,
               "flux::paged_chunk_attention: without slots page_table must have one row per request")
    else:
        _check_list(slots, torch.int64, device,
                    "flux::paged_chunk_attention: slots must be a contiguous int64 vector on the query device",
                    requests, "flux::paged_chunk_attention: slots must have one entry per request")
    if positions is not None:
        _check_list(positions, torch.int64, device,
                    "flux::paged_chunk_attention: positions must be a contiguous int64 vector on the query device",
                    requests, "flux::paged_chunk_attention: positions must have one entry per request")
    if not (key_pages.device == device and value_pages.device == device and page_table.device == device):
        _check(False, "flux::paged_chunk_attention: tensor devices must match")
    if not (key_pages.stride(3) == 1 and value_pages.stride(3) == 1 or pages[3] == 1):
        _check(False, "flux::paged_chunk_attention: pages must have unit stride along the head dimension")
    if not (0 <= window <= _MAX_KEYS and 0 <= sinks <= _MAX_KEYS):
        _check(False, "flux::paged_chunk_attention: window and sinks must be within [0, 16777216]")
    if not (_finite_fp32(scale)):
        _check(False, "flux::paged_chunk_attention: scale must be a finite FP32 value")
    if torch.is_grad_enabled():
        _grad_free("flux::paged_chunk_attention", query, key_pages, value_pages)


def _chunk_cuda(query, key_pages, value_pages, page_table, lengths, offsets, scale, window=0, sinks=0, slots=None,
                positions=None):
    _validate_chunk(query, key_pages, value_pages, page_table, lengths, offsets, scale, window, sinks, slots, positions)
    _require_gpu("flux::paged_chunk_attention", query)
    tokens, heads, dim = query.shape
    requests = offsets.shape[0] - 1
    if tokens == 0 or requests == 0:
        return query.new_zeros((tokens, heads, dim))
    pages, kv_heads, page_size, _ = key_pages.shape
    slot_count, columns = page_table.shape
    output = query.new_empty((tokens, heads, dim))
    needed = _size_from("flux_paged_chunk_attention_workspace_bytes", _TYPES[query.dtype], tokens, requests, heads, kv_heads,
                        dim, page_size, columns, window, sinks)
    workspace = query.new_empty(needed // 4, dtype=torch.float32) if needed else None
    _launch("flux_paged_chunk_attention", query.device, _TYPES[query.dtype], query.data_ptr(), key_pages.data_ptr(),
            value_pages.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), offsets.data_ptr(), _address(slots),
            _address(positions), output.data_ptr(), _address(workspace), needed, scale, tokens, requests, heads, kv_heads, dim,
            pages, page_size, slot_count, columns, page_table.stride(0), window, sinks, _three(*query.stride()),
            _three(*key_pages.stride()[:3]), _three(*value_pages.stride()[:3]))
    return output


# ---------------------------------------------------------------------------
# logits_sample

def _validate_sample(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None) -> None:
    shape, device = logits.shape, logits.device
    if not (len(shape) == 2 and 0 < shape[1] <= _MAX_VOCAB):
        _check(False, "flux::logits_sample: logits must be [rows, vocab], vocab non-empty and at most 16777216")
    if not (shape[0] <= 1 << 20 and shape[0] * (shape[1] + 1023) <= 1 << 32):
        _check(False, "flux::logits_sample: more than 1048576 rows, or rows * (vocab + 1023) beyond 4294967296")
    if not (logits.dtype in _TYPES):
        _check(False, "flux::logits_sample: logits must have dtype float32, float16 or bfloat16")
    if not (logits.stride(1) == 1 or shape[1] == 1):
        _check(False, "flux::logits_sample: logits rows must be contiguous")
    for name, values, dtype in (("uniforms", uniforms, torch.float32), ("temperature", temperature, torch.float32),
                                ("top_k", top_k, torch.int64), ("top_p", top_p, torch.float32),
                                ("min_p", min_p, torch.float32)):
        if values is None:
            continue
        if not (values.dim() == 1 and values.shape[0] == shape[0] and values.dtype is dtype and values.device == device and
                values.is_contiguous()):
            _check(False, f"flux::logits_sample: {name} must be a contiguous {str(dtype)[6:]} vector on the logits device "
                          "with one entry per row")
    if torch.is_grad_enabled():
        _grad_free("flux::logits_sample", logits, uniforms, temperature, top_p, min_p)


def _sample_cuda(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None):
    _validate_sample(logits, uniforms, temperature, top_k, top_p, min_p)
    _require_gpu("flux::logits_sample", logits)
    rows, vocab = logits.shape
    tokens = logits.new_empty(rows, dtype=torch.int64)
    probabilities = logits.new_empty(rows, dtype=torch.float32)
    if rows == 0:
        return tokens, probabilities
    needed = _size_from("flux_logits_sample_workspace_bytes", rows, vocab)
    workspace = tokens.new_empty(needed // 8) if needed else None
    _launch("flux_logits_sample", logits.device, _TYPES[logits.dtype], logits.data_ptr(), logits.stride(0),
            uniforms.data_ptr(), _address(temperature), _address(top_k), _address(top_p), _address(min_p), tokens.data_ptr(),
            probabilities.data_ptr(), rows, vocab, _address(workspace), needed)
    return tokens, probabilities


# ---------------------------------------------------------------------------
# Dispatcher registration.

_KERNELS = {
    "paged_step_layout": (_layout_cuda, _validate_layout),
    "paged_cache_write_rows": (_rows_cuda, _validate_rows_pools),
    "paged_chunk_attention": (_chunk_cuda, _validate_chunk),
    "logits_sample": (_sample_cuda, _validate_sample),
}

for _name, (_cuda, _validate) in _KERNELS.items():
    _LIBRARY.impl(_name, _cuda, "CUDA")
    _LIBRARY.impl(_name, _cpu_kernel(_name, _validate), "CPU")


@torch.library.register_fake("flux::paged_step_layout")
def _layout_fake(page_table, slots, positions, counts, page_size, tokens):
    _validate_layout(page_table, slots, positions, counts, page_size, tokens)
    return slots.new_empty((slots.shape[0] + 1,)), *(slots.new_empty((tokens,)) for _ in range(3))


@torch.library.register_fake("flux::paged_cache_write_rows")
def _rows_fake(key, value, key_pages, value_pages, rows):
    _validate_rows(key, value, key_pages, value_pages, rows)


@torch.library.register_fake("flux::paged_chunk_attention")
def _chunk_fake(query, key_pages, value_pages, page_table, lengths, offsets, scale, window=0, sinks=0, slots=None,
                positions=None):
    _validate_chunk(query, key_pages, value_pages, page_table, lengths, offsets, scale, window, sinks, slots, positions)
    return query.new_empty(query.shape)


@torch.library.register_fake("flux::logits_sample")
def _sample_fake(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None):
    _validate_sample(logits, uniforms, temperature, top_k, top_p, min_p)
    return logits.new_empty((logits.shape[0],), dtype=torch.int64), logits.new_empty((logits.shape[0],), dtype=torch.float32)


# ---------------------------------------------------------------------------
# Python entry points.

class _Overloads:
    __slots__ = STEP_OPERATOR_NAMES

    def __init__(self) -> None:
        for name in STEP_OPERATOR_NAMES:
            setattr(self, name, getattr(torch.ops.flux, name).default)


_OPS = _Overloads()


def native_paged_step_is_available() -> bool:
    return _availability("paged_step_layout", "paged_cache_write_rows", "paged_chunk_attention")


def native_logits_sample_is_available() -> bool:
    return _availability("logits_sample")


def paged_step_layout_native(page_table: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
                             counts: torch.Tensor | None, page_size: int, tokens: int
                             ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Places of a step's packed tokens; returns (offsets [requests + 1], each token's request, position and pool row).

    Request i has ``counts[i]`` (default one) tokens from ``positions[i]`` on of ``slots[i]``, as ``paged_cache_reserve``
    gave them; refused ones (position -1) have none.  ``tokens`` is the step's fixed size: entries behind the last token
    are -1, and tokens that do not fit are left out (``paged_chunk_attention`` then needs ``positions``: a request that was
    cut no longer ends with its sequence's last token).  A token beyond the table's columns or on no page has the row -1.
    """
    _ready("paged step")
    return _OPS.paged_step_layout(page_table, slots, positions, counts, page_size, tokens)


def paged_cache_write_rows_native(key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor,
                                  value_pages: torch.Tensor, rows: torch.Tensor) -> None:
    """Packed tokens' ``key``, ``value`` [T, Hkv, D] of one layer to the rows of the pool that ``paged_step_layout`` gave.

    Rows outside the pool are skipped; two tokens must not name the same row.
    """
    _ready("paged step")
    _OPS.paged_cache_write_rows(key, value, key_pages, value_pages, rows)


def paged_chunk_attention_native(query: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                                 page_table: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor, scale: float,
                                 window: int = 0, sinks: int = 0, slots: torch.Tensor | None = None,
                                 positions: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA attention of packed tokens ``query`` [T, Hq, D] over their sequences' pages, whose rows are written.

    Request i has the tokens ``offsets[i]`` to ``offsets[i + 1]`` and row ``slots[i]`` (i without slots) of ``page_table``
    and ``lengths``; its first token is at ``positions[i]`` (default: its tokens are the sequence's last).  A token sees the
    keys up to its own, with ``window`` > 0 the last ``window`` of them and the first ``sinks``.  Keys on an entry outside
    the pool are left out; tokens that see nothing, or of no request, give zeros.  ``offsets`` must not decrease.
    16-bit weights are rounded once to the type for their product with the values, as in ``window_attention`` and also
    for a single token, whose weights ``paged_decode_attention`` holds in two terms.  A call takes a workspace of up to
    138 MB at 128 dims (273 MB at 256, float32 54 MB), because the host does not know the lengths.
    """
    _ready("paged step")
    return _OPS.paged_chunk_attention(query, key_pages, value_pages, page_table, lengths, offsets, scale, window, sinks,
                                      slots, positions)


def logits_sample_native(logits: torch.Tensor, uniforms: torch.Tensor, temperature: torch.Tensor | None = None,
                         top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                         min_p: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The next token of each row of ``logits`` [rows, vocab] by ``uniforms`` in [0, 1); returns (tokens, probabilities).

    All options are vectors with an entry per row.  After division by ``temperature`` (0: greedy) the ``top_k`` largest
    logits are kept (0: all), of those the largest while the mass before them is below ``top_p``, of those the ones
    at least ``min_p`` times as probable as the largest; equal logits are kept from the lowest index on.  The token is the
    first, by index, at which the kept mass exceeds ``uniforms`` times all of it; its probability is its share.  No rows (a step
    in which no prompt ends) give empty results.
    """
    _ready("logits sample")
    return _OPS.logits_sample(logits, uniforms, temperature, top_k, top_p, min_p)
