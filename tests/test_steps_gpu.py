"""GPU parity of the operators of mixed steps against plain forms (``oracle/steps.py``).

What moves or counts is exact, and so are sampled tokens: weights that are held in integers of 2^-45 or finer move a border
between tokens by less than 1e-9 of the mass, and no case's random number is that close to one.  Attention's tolerances are
computed from the inputs (``oracle.serving.attention_bound``).
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from flux_amd import ops
from oracle import serving as ref
from oracle import steps

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _close(actual, expected, bound):
    error = (actual.cpu().double() - expected).abs()
    beyond = float((error - bound).nan_to_num(nan=math.inf).max())
    assert beyond <= 0, f"off by {beyond:.3g} beyond the bound, at most {float(error.max()):.3g}"


def _to(values, device):
    return {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in values.items()}


# --------------------------------------------------------------------------- layout

def _layout_case(seed, requests, slots, columns, page_size, longest):
    g = torch.Generator().manual_seed(seed)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=g)

    return {"page_table": whole(-2, 500, slots, columns).to(torch.int32), "slots": whole(-1, slots + 1, requests),
            "positions": whole(-3, columns * page_size + 5, requests), "counts": whole(-1, longest, requests),
            "page_size": page_size}


@pytest.mark.parametrize("requests", [1, 2, 5, 63, 64, 65, 1000, 1023, 1024, 1025, 3100])
@pytest.mark.parametrize("tokens", [1, 7, 64, 1023, 1024, 1025, 5000])
def test_step_layout(gpu_device, requests, tokens):
    case = _layout_case(requests + tokens, requests, 40, 9, 7, 12)
    actual = ops.paged_step_layout_native(**_to(case, gpu_device), tokens=tokens)
    for a, e in zip(actual, steps.step_layout(**case, tokens=tokens)):
        assert a.dtype == torch.int64 and a.tolist() == e


def test_step_layout_lists_and_extremes(gpu_device):
    case = _layout_case(3, 30, 20, 5, 16, 200)
    # One token each; a table inside a wider one; counts that no step holds; positions at the end of 64 bits.
    expected = steps.step_layout(**{**case, "counts": None}, tokens=50)
    device = _to(case, gpu_device)
    assert [a.tolist() for a in ops.paged_step_layout_native(**{**device, "counts": None}, tokens=50)] == list(expected)
    wide = torch.full((20, 40), 77, dtype=torch.int32, device=gpu_device)
    wide[:, 3:8] = device["page_table"]
    device["page_table"] = wide[:, 3:8]
    for a, e in zip(ops.paged_step_layout_native(**device, tokens=900), steps.step_layout(**case, tokens=900)):
        assert a.tolist() == e
    case["counts"] = torch.full((30,), 1 << 62)
    case["slots"], case["positions"] = torch.arange(30) % 20, torch.arange(30)
    offsets, request, position, row = ops.paged_step_layout_native(**_to(case, gpu_device), tokens=2000)
    assert offsets.tolist() == [0] + [2000] * 30 and set(request.tolist()) == {0}
    assert position.tolist() == list(range(2000)) and row[80:].tolist() == [-1] * 1920
    case["counts"], case["positions"] = torch.ones(30, dtype=torch.int64), torch.full((30,), 2 ** 63 - 1)
    _, request, position, row = ops.paged_step_layout_native(**_to(case, gpu_device), tokens=31)
    assert request.tolist() == [*range(30), -1] and position.tolist() == [2 ** 63 - 1] * 30 + [-1] and set(row.tolist()) == {-1}
    none = torch.empty(0, dtype=torch.int64, device=gpu_device)
    empty = ops.paged_step_layout_native(case["page_table"].to(gpu_device), none, none, None, 16, 3)
    assert [a.tolist() for a in empty] == [[0], [-1] * 3, [-1] * 3, [-1] * 3]
    assert [a.tolist() for a in ops.paged_step_layout_native(**_to(case, gpu_device), tokens=0)][1:] == [[], [], []]


# --------------------------------------------------------------------------- rows

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dim,page_size,tokens", [(3, 64, 16, 1), (3, 64, 16, 16), (3, 64, 16, 17), (8, 128, 64, 100),
                                                        (1, 1, 5, 33), (2, 5, 3, 200), (5, 80, 48, 77)])
def test_write_rows(gpu_device, dtype, heads, dim, page_size, tokens):
    g = torch.Generator().manual_seed(tokens)
    pages = tokens // page_size + 4
    pools = [torch.randn(pages, heads, page_size, dim, generator=g).to(dtype) for _ in range(2)]
    packed = torch.randn(tokens, 2 * heads + 1, dim, generator=g).to(dtype)
    key, value = packed[:, 1 : heads + 1], packed[:, heads + 1 :]
    rows = torch.randperm(pages * page_size, generator=g)[:tokens]
    rows[::5] = torch.tensor([-1, pages * page_size, -(2 ** 62), 2 ** 62])[torch.arange(len(rows[::5])) % 4]
    device = [t.to(gpu_device) for t in pools]
    moved = packed.to(gpu_device)
    steps.write_rows(key, value, *pools, rows)
    ops.paged_cache_write_rows_native(moved[:, 1 : heads + 1], moved[:, heads + 1 :], *device, rows.to(gpu_device))
    assert all(torch.equal(a.cpu(), e) for a, e in zip(device, pools))
    # Pages with heads inside, in a store that leaves the rows at no 16 bytes.
    stores = [torch.zeros(pages, page_size, heads, dim + 3, device=gpu_device, dtype=dtype) for _ in range(2)]
    views = [t[..., 1 : dim + 1].transpose(1, 2) for t in stores]
    ops.paged_cache_write_rows_native(moved[:, 1 : heads + 1], moved[:, heads + 1 :], *views, rows.to(gpu_device))
    plain = [torch.zeros_like(t) for t in pools]
    steps.write_rows(key, value, *plain, rows)
    assert all(torch.equal(a.cpu(), e) for a, e in zip(views, plain))
    assert not any(bool(t[..., 0].any() or t[..., dim + 1 :].any()) for t in stores)
    none = torch.empty(0, dtype=torch.int64, device=gpu_device)
    ops.paged_cache_write_rows_native(moved[:0, 1 : heads + 1], moved[:0, heads + 1 :], *device, none)
    assert all(torch.equal(a.cpu(), e) for a, e in zip(device, pools))


# --------------------------------------------------------------------------- chunk attention

def _chunk_case(seed, dtype, heads, kv_heads, dim, page_size, spans, spare_rows=0, spare_pages=3, scale=None):
    """CPU tensors of requests (tokens, earlier keys) whose pages lie scattered in the pool; what no sequence holds is NaN."""
    g = torch.Generator().manual_seed(seed)
    lengths = [c + b for c, b in spans]
    columns = max(1, -(-max([*lengths, 1]) // page_size))
    needed = [-(-n // page_size) for n in lengths]
    pages = sum(needed) + spare_pages
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(spans), columns), -1, dtype=torch.int32)
    key_pages, value_pages = (torch.full((pages, kv_heads, page_size, dim), math.nan, dtype=dtype) for _ in range(2))
    for b, n in enumerate(lengths):
        for c in range(needed[b]):
            page, rows = order.pop(), min(page_size, n - c * page_size)
            table[b, c] = page
            key_pages[page, :, :rows] = torch.randn(kv_heads, rows, dim, generator=g).to(dtype)
            value_pages[page, :, :rows] = torch.randn(kv_heads, rows, dim, generator=g).to(dtype)
    tokens = sum(c for c, _ in spans) + spare_rows
    offsets = torch.tensor([0, *(c for c, _ in spans)]).cumsum(0)
    return {"query": torch.randn(tokens, heads, dim, generator=g).to(dtype), "key_pages": key_pages, "value_pages": value_pages,
            "page_table": table, "lengths": torch.tensor(lengths), "offsets": offsets, "scale": scale or dim ** -0.5}


def _bound(case, expected):
    terms = int(min(int(case["lengths"].max()), case["page_table"].shape[1] * case["key_pages"].shape[2]))
    return ref.attention_bound(case["query"], case["key_pages"].nan_to_num(), case["value_pages"].nan_to_num(), case["scale"],
                               max(terms, 1), case["query"].dtype, expected, rounded_weights=True)


def _check_chunk(case, device, actual=None, **options):
    expected = steps.chunk_attention(**case, **options)
    if actual is None:
        actual = ops.paged_chunk_attention_native(**_to(case, device), **_to(options, device))
    assert actual.dtype == case["query"].dtype and actual.is_contiguous() and actual.shape == expected.shape
    _close(actual, expected, _bound(case, expected))
    return actual


SPANS = [(1, 0), (0, 40), (5, 0), (1, 15), (16, 16), (1, 300), (33, 100), (0, 0), (70, 1), (3, 64), (17, 130)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,page_size", [(64, 16), (128, 64), (256, 16), (80, 48), (72, 7), (40, 1), (100, 5), (5, 3),
                                           (1, 4), (192, 100), (33, 16)])
def test_chunk_heads_and_pages(gpu_device, dtype, dim, page_size):
    for heads, kv_heads in ((9, 3), (2, 2), (20, 1)):
        case = _chunk_case(dim + page_size, dtype, heads, kv_heads, dim, page_size, SPANS, spare_rows=9)
        out = _check_chunk(case, gpu_device)
        assert not out[-9:].any()


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 9), (1, 0), (1, 1), (16, 0), (31, 4), (32, 33), (100, 1), (150, 64),
                                          (1000, 5), (1 << 24, 1 << 24)])
@pytest.mark.parametrize("dtype,dim,page_size", [(torch.float32, 64, 16), (torch.bfloat16, 128, 24),
                                                 (torch.float16, 256, 33), (torch.float16, 64, 16)])
def test_chunk_windows(gpu_device, dtype, dim, page_size, window, sinks):
    case = _chunk_case(7, dtype, 6, 2, dim, page_size, [(1, 0), (40, 0), (1, 256), (50, 350), (130, 3), (2, 99)])
    _check_chunk(case, gpu_device, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(torch.float32, 9, 3, 64), (torch.bfloat16, 4, 1, 128),
                                                      (torch.float16, 2, 2, 64), (torch.bfloat16, 2, 1, 200),
                                                      (torch.float32, 2, 1, 128), (torch.float32, 2, 1, 256)])
def test_chunk_of_every_length(gpu_device, dtype, heads, kv_heads, dim):
    """Tiles that end anywhere, prompts from their start."""
    for count in [*range(1, 20), 31, 32, 33, 42, 43, 63, 64, 65, 127, 128, 129, 130]:
        for before in (0, 61):
            _check_chunk(_chunk_case(count, dtype, heads, kv_heads, dim, 16, [(count, before)]), gpu_device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (3000, 70)])
def test_chunk_long_keys_are_cut(gpu_device, dtype, window, sinks):
    """Few tokens over long keys next to short requests: their tiles are cut and joined."""
    spans = [(2, 9000), (3, 0), (1, 5000), (0, 2000), (37, 4321), (1, 700), (90, 0)]
    _check_chunk(_chunk_case(5, dtype, 3, 1, 64, 16, spans, spare_rows=5), gpu_device, window=window, sinks=sinks)
    _check_chunk(_chunk_case(6, dtype, 2, 1, 128, 48, [(4, 8000)]), gpu_device, window=window, sinks=sinks)
    _check_chunk(_chunk_case(8, dtype, 1, 1, 160, 32, [(1, 6000), (9, 3000)]), gpu_device, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
def test_chunk_many_requests(gpu_device, dtype):
    """More requests than one round's threads, in no order of lengths, empty ones among them."""
    rng = random.Random(2)
    spans = [(rng.choice((0, 1, 1, 1, 2, 9)), rng.choice((0, 1, 5, 40, 90, 600))) for _ in range(601)]
    spans[0] = spans[300] = (0, 0)
    _check_chunk(_chunk_case(3, dtype, 2, 2, 32, 8, spans, spare_rows=3), gpu_device)


def test_chunk_slots_positions_and_bad_pages(gpu_device):
    for dtype in TYPES:
        case = _chunk_case(13, dtype, 6, 2, 64, 16, [(4, 46), (150, 50), (3, 30), (20, 100), (7, 0), (2, 5)])
        # Rows in another order, twice, and outside the table; positions in the middle, before and behind the keys.
        slots = torch.tensor([2, 1, 6, 0, 3, -1])
        _check_chunk(case, gpu_device, slots=slots)
        _check_chunk(case, gpu_device, slots=slots, positions=torch.tensor([0, 190, 3, 60, 117, 0]))
        _check_chunk(case, gpu_device, slots=torch.tensor([1, 1, 1, 3, 3, 0]),
                     positions=torch.tensor([-2, 10, 2 ** 62, -(2 ** 62), 100, 2 ** 63 - 1]))
        # Lengths beyond the columns and negative ones.
        case["key_pages"], case["value_pages"] = case["key_pages"].nan_to_num(), case["value_pages"].nan_to_num()
        case["lengths"] = torch.tensor([1 << 40, 200, -5, 120, 7, 7])
        _check_chunk(case, gpu_device)
        # Entries outside the pool are left out: the tokens attend over the others.
        case["lengths"] = torch.tensor([50, 200, 33, 120, 7, 7])
        case["page_table"][0, 1] = -1
        case["page_table"][1, 3] = case["key_pages"].shape[0]
        case["page_table"][1, 4] = 2 ** 31 - 1
        case["page_table"][2] = -7
        case["page_table"][3, 0] = -1
        case["key_pages"][0], case["value_pages"][0] = math.nan, math.inf  # what a row that is left out must not read
        case["page_table"][case["page_table"] == 0] = -1
        out = _check_chunk(case, gpu_device)
        assert not out[154:157].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_chunk_strides_and_alignment(gpu_device, dtype):
    for dim in (64, 80):
        case = _chunk_case(17, dtype, 6, 2, dim, 16, [(4, 46), (50, 150), (1, 300), (20, 10)])
        device = _to(case, gpu_device)
        expected = ops.paged_chunk_attention_native(**device)
        _check_chunk(case, gpu_device, expected)
        # [P, page, heads, D] pages, a table inside a wider one, a query inside a packed projection, another dim stride.
        moved = dict(device)
        for name in ("key_pages", "value_pages"):
            moved[name] = device[name].transpose(1, 2).contiguous().transpose(1, 2)
        wide = torch.full((4, 40), 99, dtype=torch.int32, device=gpu_device)
        wide[:, 3 : 3 + device["page_table"].shape[1]] = device["page_table"]
        moved["page_table"] = wide[:, 3 : 3 + device["page_table"].shape[1]]
        packed = torch.randn(75, 10, dim, device=gpu_device).to(dtype)
        packed[:, 2:8] = device["query"]
        moved["query"] = packed[:, 2:8]
        assert torch.equal(ops.paged_chunk_attention_native(**moved), expected)
        moved["query"] = device["query"].transpose(0, 2).contiguous().transpose(0, 2)
        assert torch.equal(ops.paged_chunk_attention_native(**moved), expected)
        # Rows that start at no 16 bytes.
        for name in ("key_pages", "value_pages"):
            store = torch.randn(*device[name].shape[:3], dim + 3, device=gpu_device).to(dtype)
            store[..., 1 : dim + 1] = device[name]
            moved[name] = store[..., 1 : dim + 1]
        _check_chunk(case, gpu_device, ops.paged_chunk_attention_native(**moved))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page_size", [(200, 1, 16, 1), (130, 2, 72, 1000), (257, 1, 64, 17), (64, 64, 8, 3)])
def test_chunk_wide_groups_and_odd_pages(gpu_device, dtype, heads, kv_heads, dim, page_size):
    """Groups beyond a tile's rows, many KV heads, pages of one row and pages beyond every length."""
    case = _chunk_case(97, dtype, heads, kv_heads, dim, page_size, [(3, 50), (1, 700), (0, 5), (20, 0)], spare_rows=2)
    _check_chunk(case, gpu_device)
    _check_chunk(case, gpu_device, window=33, sinks=2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [0, 40, 1 << 24])
def test_chunk_tables_of_the_largest_width(gpu_device, dtype, window):
    case = _chunk_case(101, dtype, 4, 2, 64, 16, [(3, 50), (1, 700), (80, 100)])
    device = _to(case, gpu_device)
    wide = torch.full((3, (1 << 24) // 16), -1, dtype=torch.int32, device=gpu_device)
    wide[:, : case["page_table"].shape[1]] = device["page_table"]
    out = ops.paged_chunk_attention_native(**{**device, "page_table": wide}, window=window, sinks=window)
    _check_chunk(case, gpu_device, out, window=window, sinks=window)


@pytest.mark.parametrize("dtype", TYPES)
def test_chunk_offsets_that_decrease(gpu_device, dtype):
    """Not allowed, and within bounds all the same."""
    case = _chunk_case(103, dtype, 4, 2, 64, 16, [(10, 3000), (40, 600), (30, 100)])
    device = _to(case, gpu_device)
    for offsets in ([0, 50, 10, 80], [80, 0, 80, 0], [-5, 2 ** 62, -(2 ** 62), 80], [70, 60, 50, 40]):
        device["offsets"] = torch.tensor(offsets, device=gpu_device)
        assert ops.paged_chunk_attention_native(**device).shape == case["query"].shape
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 80, 128])
def test_chunk_infinities_and_nan(gpu_device, dtype, dim):
    """They reach the tokens that see them, and no others; scores of -inf weigh nothing."""
    case = _chunk_case(19, dtype, 4, 2, dim, 16, [(20, 60), (2, 3000), (1, 100)])
    table = case["page_table"]
    case["value_pages"][table[0, 4], 0, 10] = math.nan       # key 74: the request's last six tokens see it
    case["value_pages"][table[1, 50], 1, 3, 0] = math.inf
    case["key_pages"][table[2, 2], :, 5] = math.nan
    expected = steps.chunk_attention(**case)
    actual = ops.paged_chunk_attention_native(**_to(case, gpu_device)).cpu().double()
    assert torch.equal(actual.isnan(), expected.isnan()) and torch.equal(actual == math.inf, expected == math.inf)
    finite = expected.isfinite()
    assert bool(finite[:14].all()) and not bool(finite[14:20, :2].any()) and not bool(finite[22].any())
    clean = {**case, "key_pages": case["key_pages"].nan_to_num(posinf=0), "value_pages": case["value_pages"].nan_to_num(posinf=0)}
    bound = _bound(clean, expected.nan_to_num(posinf=0))
    assert float(((actual - expected).abs() - bound)[finite].max()) <= 0
    # Every score of the first request is -inf, and every second one of the others.
    case = _chunk_case(23, dtype, 4, 2, dim, 16, [(20, 60), (2, 3000)])
    case["query"][..., 0] = 1
    key = case["key_pages"]
    key[case["page_table"][0, :5].long(), :, :, 0] = -math.inf
    key[:, :, ::2, 0] = -math.inf
    expected = steps.chunk_attention(**case)
    actual = ops.paged_chunk_attention_native(**_to(case, gpu_device))
    assert bool(expected.isfinite().all())
    bounded = {**case, "key_pages": key.nan_to_num(neginf=0)}
    _close(actual, expected, _bound(bounded, expected))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.125, 1e-38, 1e38, 3e38, -3e38, 1e-45])
def test_chunk_scales(gpu_device, dtype, scale):
    """Scales of either sign and next to what float32 holds, on scores that stay finite."""
    case = _chunk_case(29, dtype, 2, 1, 64, 16, [(20, 60), (2, 3000)], scale=scale)
    if abs(scale) > 1:  # scores of -1, 0 and 1 times a power of two below the largest float
        case["query"].zero_()[..., 0] = 1
        case["key_pages"][..., 1:] = 0
        case["key_pages"][..., 0] = case["key_pages"][..., 0].sign()
    expected = steps.chunk_attention(**case)
    actual = ops.paged_chunk_attention_native(**_to(case, gpu_device))
    bounded = {**case, "scale": scale if abs(scale) < 1 else 0.0}  # the scores are exact, and their differences 0 or huge
    _close(actual, expected, _bound(bounded, expected))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 15])
def test_chunk_scores_far_from_zero(gpu_device, dtype, size):
    """Scores about 2^24 and 2^30, exact and as far apart as a few: every key counts."""
    case = _chunk_case(37, dtype, 2, 1, 64, 16, [(20, 60), (2, 3000)], scale=1.0)
    case["query"].zero_()[..., 0] = size
    case["query"][..., 1] = 1
    key = case["key_pages"]
    key[..., 2:] = 0
    key[..., 1] = (key[..., 1] * 4 / size).round() * size
    key[..., 0] = size
    key[..., 1] = torch.where(key[..., 1].abs() < 1, key[..., 1], key[..., 1].sign() * 128)  # a step of 2^30 is 64
    expected = steps.chunk_attention(**case)
    actual = ops.paged_chunk_attention_native(**_to(case, gpu_device))
    _close(actual, expected, _bound({**case, "scale": 0.0}, expected))


def test_chunk_scale_zero(gpu_device):
    for dtype in TYPES:
        case = {**_chunk_case(31, dtype, 2, 1, 64, 16, [(20, 60), (2, 3000)]), "scale": 0.0}
        _check_chunk(case, gpu_device)


# Inputs whose results tell every key: as in the tests of the serving operators.

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 1, 64), (20, 1, 128), (4, 2, 80), (2, 1, 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2000, 40)])
def test_chunk_loses_no_key(gpu_device, dtype, heads, kv_heads, dim, window, sinks):
    spans, page_size = [(2, 9000), (40, 0), (1, 700), (30, 5000), (1, 15), (130, 200)], 48
    case = _chunk_case(67, dtype, heads, kv_heads, dim, page_size, spans, scale=math.log(2))
    case["query"].zero_()[..., 0] = (1 + torch.arange(heads) % 2).to(dtype)
    for b, (count, before) in enumerate(spans):
        for c in range(-(-(count + before) // page_size)):
            page, tile = int(case["page_table"][b, c]), torch.arange(c * page_size, (c + 1) * page_size) // 16
            case["key_pages"][page], case["value_pages"][page] = 0, 0
            case["key_pages"][page, :, :, 0] = -(tile % 8).to(dtype)
            case["value_pages"][page, :, torch.arange(page_size), tile % dim] = 1
    expected = steps.chunk_attention(**case, window=window, sinks=sinks)
    # Relative, as all terms are positive: the exponents, at most 32 below the maximum, are off by less than 2^-17 of the weight
    # together with the maximum's steps, the exponentials by as much, what is left of a power of two in 16 bits by as much
    # again; 9002 / 4 additions one after the other by 2^-24 each, in both sums, and the quotient; the result is rounded once.
    relative = 2.0 ** -15 + 2300 * 2.0 ** -23 + torch.finfo(dtype).eps / 2
    bound = relative * expected + torch.finfo(dtype).tiny
    _close(ops.paged_chunk_attention_native(**_to(case, gpu_device), window=window, sinks=sinks), expected, bound)
    # The bound tells a lost tile of 16 keys of the longest sequence, wherever it lies.
    keys = torch.zeros(9002, dim, dtype=torch.float64), torch.zeros(9002, dim, dtype=torch.float64)
    keys[0][:, 0] = -(torch.arange(9002) // 16 % 8).double()
    keys[1][torch.arange(9002), torch.arange(9002) // 16 % dim] = 1
    seen = ref.visible_keys(9001, 9002, window, sinks)
    for first in {seen[0], seen[len(seen) // 2] // 16 * 16, 9001 // 16 * 16}:
        kept = [j for j in seen if not first <= j < first + 16]
        lost = ref.attend(case["query"][1, 0], keys[0][kept], keys[1][kept], case["scale"])
        assert bool(((lost - expected[1, 0]).abs() > bound[1, 0]).any())


# float32 chunks of many rows are multiplied in three limbs of 16 bits: 141 tokens of 16 heads are such.

MANY = [(70, 60), (2, 3000), (60, 700), (9, 0)]


def _many_rows(seed, dim=64, scale=None):
    return _chunk_case(seed, torch.float32, 16, 1, dim, 16, MANY, scale=scale)


@pytest.mark.parametrize("dim", [64, 40, 33, 2])
@pytest.mark.parametrize("window,sinks", [(0, 0), (900, 20), (1, 0)])
def test_chunk_of_many_rows(gpu_device, dim, window, sinks):
    case = _many_rows(71, dim)
    _check_chunk(case, gpu_device, window=window, sinks=sinks)
    moved = _to(case, gpu_device)
    for name in ("key_pages", "value_pages"):  # rows that start at no 16 bytes
        store = torch.full((*moved[name].shape[:3], dim + 3), math.nan, device=gpu_device)
        store[..., 1 : dim + 1] = moved[name]
        moved[name] = store[..., 1 : dim + 1]
    moved["query"] = moved["query"].transpose(0, 2).contiguous().transpose(0, 2)
    _check_chunk(case, gpu_device, ops.paged_chunk_attention_native(**moved, window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("name,factor", [("value_pages", 2.0 ** 21), ("value_pages", 2.0 ** -70), ("value_pages", 2.0 ** -110),
                                         ("query", 2.0 ** 64), ("query", 2.0 ** -60), ("key_pages", 2.0 ** 70),
                                         ("key_pages", 2.0 ** -90)])
def test_chunk_of_many_rows_and_magnitudes(gpu_device, name, factor):
    """What the limbs do not hold is computed otherwise; every second request has ordinary numbers."""
    case = _many_rows(73)
    if name == "query":
        case["query"][:70] *= factor
    else:
        case[name][case["page_table"][0, :9].long()] *= factor
    if factor > 1 and name != "value_pages":  # the scores stay as they were
        case["scale"] /= factor
    expected = steps.chunk_attention(**case)
    actual = ops.paged_chunk_attention_native(**_to(case, gpu_device))
    for rows, pages in ((slice(0, 70), case["page_table"][0, :9]), (slice(70, 141), case["page_table"][1:].flatten())):
        pages = pages[pages >= 0].long()
        own = {**case, "query": case["query"][rows], "key_pages": case["key_pages"][pages], "value_pages": case["value_pages"][pages]}
        _close(actual[rows], expected[rows], _bound(own, expected[rows]))


@pytest.mark.parametrize("scale", [-0.125, 1e-38, 1e38, -3e38, 1e-45])
def test_chunk_of_many_rows_and_scales(gpu_device, scale):
    case = _many_rows(79, scale=scale)
    if abs(scale) > 1:
        case["query"].zero_()[..., 0] = 1
        case["key_pages"][..., 1:] = 0
        case["key_pages"][..., 0] = case["key_pages"][..., 0].sign()
    expected = steps.chunk_attention(**case)
    actual = ops.paged_chunk_attention_native(**_to(case, gpu_device))
    _close(actual, expected, _bound({**case, "scale": scale if abs(scale) < 1 else 0.0}, expected))


def test_chunk_of_many_rows_infinities_and_nan(gpu_device):
    case = _many_rows(83)
    table = case["page_table"]
    case["value_pages"][table[0, 4], 0, 10] = math.nan   # key 74, which the tokens 14 and on of the first request see
    case["value_pages"][table[1, 50], 0, 3, 0] = math.inf
    case["key_pages"][table[2, 2], 0, 5] = math.nan
    expected = steps.chunk_attention(**case)
    actual = ops.paged_chunk_attention_native(**_to(case, gpu_device)).cpu().double()
    assert torch.equal(actual.isnan(), expected.isnan()) and torch.equal(actual == math.inf, expected == math.inf)
    finite = expected.isfinite()
    assert bool(finite[:14].all()) and not bool(finite[14:70].any()) and not bool(finite[72:132].any()) and bool(finite[132:].all())
    clean = {**case, "key_pages": case["key_pages"].nan_to_num(posinf=0), "value_pages": case["value_pages"].nan_to_num(posinf=0)}
    assert float(((actual - expected).abs() - _bound(clean, expected.nan_to_num(posinf=0)))[finite].max()) <= 0


@pytest.mark.parametrize("dtype", TYPES)
def test_chunk_pools_beyond_four_gigabytes(gpu_device, dtype):
    """Pages whose rows lie behind 2^32 bytes (2^31 elements): rows are written there and attended over."""
    case = _chunk_case(89, dtype, 16, 1, 64, 16, [(70, 60), (2, 3000), (80, 100)])
    pages, here = (2 ** 31) // 1024 + 4, case["key_pages"].shape[0]
    order = torch.cat((torch.arange(2), torch.arange(pages - here + 2, pages)))
    pools = [torch.empty(pages, 1, 16, 64, device=gpu_device, dtype=dtype) for _ in range(2)]
    rows = (order[:, None] * 16 + torch.arange(16)).flatten().to(gpu_device)
    key, value = (case[n].transpose(1, 2).reshape(-1, 1, 64).to(gpu_device) for n in ("key_pages", "value_pages"))
    ops.paged_cache_write_rows_native(key, value, *pools, rows)
    table = case["page_table"]
    far = {**case, "key_pages": pools[0], "value_pages": pools[1], "page_table": torch.where(table >= 0, order[table.long().clamp(min=0)], -1).int()}
    _check_chunk(case, gpu_device, ops.paged_chunk_attention_native(**_to(far, gpu_device)))


def test_chunk_no_tokens_or_requests(gpu_device):
    case = _to(_chunk_case(3, torch.bfloat16, 4, 2, 64, 16, [(3, 5)]), gpu_device)
    nothing = torch.zeros(1, dtype=torch.int64, device=gpu_device)
    assert not ops.paged_chunk_attention_native(**{**case, "offsets": nothing}).any()
    assert ops.paged_chunk_attention_native(**{**case, "query": case["query"][:0]}).shape == (0, 4, 64)
    # Offsets beyond the tokens are cut; the positions stay those of the whole request.
    short = ops.paged_chunk_attention_native(**{**case, "query": case["query"][:2].contiguous()})
    assert torch.equal(short, ops.paged_chunk_attention_native(**case)[:2])
    # None of the requests has a token.
    zeros = torch.zeros(2, dtype=torch.int64, device=gpu_device)
    assert not ops.paged_chunk_attention_native(**{**case, "offsets": zeros}).any()
    # Rows before the first request are of none.
    later = {**case, "query": torch.cat((case["query"], case["query"])), "offsets": case["offsets"] + 3}
    out = ops.paged_chunk_attention_native(**later)
    assert not out[:3].any() and torch.equal(out[3:], ops.paged_chunk_attention_native(**case))


# --------------------------------------------------------------------------- sampling

def _check_sample(logits, device, **options):
    tokens, probabilities = steps.sample(logits, **options)
    actual, shares = ops.logits_sample_native(logits.to(device), **_to(options, device))
    assert actual.dtype == torch.int64 and shares.dtype == torch.float32
    assert actual.tolist() == tokens
    # Weights and their sum are off by at most 2^-37 of 1 each (2^24 tokens have 38 bits), the share is rounded to float32.
    expected = torch.tensor(probabilities, dtype=torch.float64)
    assert float(((shares.cpu().double() - expected).abs() - (2.0 ** -24 + 2.0 ** -36) * expected - 2.0 ** -149).max()) <= 0
    return actual


def _options(g, rows, share=0.6):
    def some(values, off):
        return torch.where(torch.rand(rows, generator=g) < share, values, off)

    return {"uniforms": torch.rand(rows, generator=g), "temperature": 0.3 + 1.5 * torch.rand(rows, generator=g),
            "top_k": some(torch.randint(1, 300, (rows,), generator=g), torch.tensor(0)),
            "top_p": some(torch.rand(rows, generator=g), torch.tensor(1.0)),
            "min_p": some(0.2 * torch.rand(rows, generator=g), torch.tensor(0.0))}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 64, 1000, 1023, 1024, 1025, 4099, 49152])
def test_sample_filters(gpu_device, dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    rows = 24 if vocab < 10000 else 2
    logits = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    _check_sample(logits, gpu_device, **_options(g, rows))
    only = _options(g, rows)
    _check_sample(logits, gpu_device, uniforms=only["uniforms"])
    for name in ("temperature", "top_k", "top_p", "min_p"):
        _check_sample(logits, gpu_device, uniforms=only["uniforms"], **{name: only[name]})


@pytest.mark.parametrize("rows,vocab", [(1, 128000), (3, 200003), (300, 517)])
def test_sample_shapes(gpu_device, rows, vocab):
    g = torch.Generator().manual_seed(rows)
    _check_sample((2 * torch.randn(rows, vocab, generator=g)).bfloat16(), gpu_device, **_options(g, rows))


def test_sample_reaches_every_token(gpu_device):
    """A number between each token's borders gives it, for every token that is kept, and no other."""
    g = torch.Generator().manual_seed(5)
    row = torch.randn(40, generator=g)
    for options in ({}, {"top_k": 7}, {"top_p": 0.8}, {"min_p": 0.3}, {"top_k": 20, "top_p": 0.7, "min_p": 0.05}):
        weight = torch.exp(row.double() - row.double().max())
        order = torch.argsort(row, descending=True)
        kept = order[: options.get("top_k", 40)]
        mass = weight[kept]
        kept = kept[(mass.cumsum(0) - mass < options.get("top_p", 1.0) * mass.sum()) & (mass >= options.get("min_p", 0.0))]
        kept = kept.sort().values
        reached = weight[kept].cumsum(0) / weight[kept].sum()
        middle = ((reached + torch.cat((torch.zeros(1), reached[:-1]))) / 2).float()
        rows = len(kept)
        vectors = {k: torch.full((rows,), v, dtype=torch.int64 if k == "top_k" else torch.float32) for k, v in options.items()}
        actual = _check_sample(row.expand(rows, 40).contiguous(), gpu_device, uniforms=middle, **vectors)
        assert actual.tolist() == kept.tolist()


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_ties(gpu_device, dtype):
    """Equal logits are kept from the lowest index on."""
    g = torch.Generator().manual_seed(9)
    logits = torch.randint(0, 4, (64, 5000), generator=g).to(dtype)
    logits[5:9] = 0.25  # all equal
    logits[9, ::2] = -0.0
    logits[9, 1::2] = 0.0
    _check_sample(logits, gpu_device, **_options(g, 64, share=0.8))
    rows = torch.arange(64)
    _check_sample(logits, gpu_device, uniforms=torch.full((64,), 1 - 2.0 ** -24), top_k=rows + 1200)
    _check_sample(logits, gpu_device, uniforms=torch.full((64,), 0.999), top_p=(rows + 1) / 70)
    _check_sample(logits, gpu_device, uniforms=torch.rand(64, generator=g), min_p=torch.full((64,), 1.0))


def test_sample_borders_of_the_options(gpu_device):
    g = torch.Generator().manual_seed(11)
    logits = 3 * torch.randn(12, 300, generator=g)
    inf, nan = math.inf, math.nan
    u = torch.tensor([0.0, -1.0, 1 - 2.0 ** -24, 1.0, 2.0, nan, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5])
    expected = u.clone()
    expected[3:5] = 1 - 2.0 ** -24  # the last token either way, unless its share is below 2^-24
    tokens, _ = steps.sample(logits, expected)
    logits[:, 299] = 5  # so that it is not
    _check_sample(logits, gpu_device, uniforms=torch.where(u > 1 - 2.0 ** -24, 1 - 2.0 ** -24, u.nan_to_num(nan=0.0)))
    actual, _ = ops.logits_sample_native(logits.to(gpu_device), u.to(gpu_device))
    assert actual.tolist() == steps.sample(logits, torch.where(u > 1 - 2.0 ** -24, 1 - 2.0 ** -24, u.nan_to_num(nan=0.0)))[0]
    half = torch.full((12,), 0.5)
    greedy = logits.argmax(1).tolist()
    for t in (0.0, -0.0, -1.0, nan, -inf):
        assert _check_sample(logits, gpu_device, uniforms=half, temperature=torch.full((12,), t)).tolist() == greedy
    _check_sample(logits, gpu_device, uniforms=half, temperature=torch.tensor([inf, 1e30, 1e-30, 1e-45, 3e38, 1e-3] * 2))
    _check_sample(logits, gpu_device, uniforms=half, top_k=torch.tensor([0, -1, 1, 2, 299, 300, 301, 2 ** 62, -(2 ** 62), 5, 6, 7]))
    assert _check_sample(logits, gpu_device, uniforms=half, top_p=torch.tensor([0.0, -1.0, 1e-30, -inf] * 3)).tolist() == greedy
    _check_sample(logits, gpu_device, uniforms=half, top_p=torch.tensor([1.0, 2.0, inf, nan, 1 - 2.0 ** -24, 0.999999] * 2))
    _check_sample(logits, gpu_device, uniforms=half, min_p=torch.tensor([0.0, -1.0, nan, 1.0, 2.0, inf, 1e-30, 1e-45, 0.5, 0.1, 0.9, 0.99]))


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_infinities_and_nan(gpu_device, dtype):
    """Masked tokens are never drawn; a row whose largest logit is not finite is greedy."""
    inf, nan = math.inf, math.nan
    g = torch.Generator().manual_seed(13)
    logits = (2 * torch.randn(9, 700, generator=g)).to(dtype)
    logits[0, ::2] = -inf
    logits[1, :699] = -inf
    logits[2] = -inf
    logits[3, 20], logits[3, 30] = inf, inf
    logits[4, 40], logits[4, 41] = nan, inf
    logits[5] = torch.finfo(dtype).min
    logits[5, 7:9] = -inf
    logits[6] = torch.finfo(dtype).min
    logits[6, 50] = torch.finfo(dtype).max
    logits[7, 1:] = -inf
    options = _options(g, 9)
    tokens = _check_sample(logits, gpu_device, **options)
    assert tokens[1:5].tolist() == [699, 0, 20, 40] and tokens[6:8].tolist() == [50, 0]
    logits[4, 40] = -nan
    assert int(_check_sample(logits, gpu_device, **options)[4]) == 40
    _check_sample(logits, gpu_device, uniforms=options["uniforms"], temperature=torch.full((9,), inf))


def test_sample_strides(gpu_device):
    g = torch.Generator().manual_seed(17)
    logits = 3 * torch.randn(6, 1003, generator=g)
    options = _options(g, 6)
    for dtype in TYPES:
        expected = _check_sample(logits.to(dtype), gpu_device, **options)
        for left in (1, 2, 8):
            store = torch.full((6, 1200), math.nan, device=gpu_device, dtype=dtype)
            store[:, left : left + 1003] = logits.to(dtype)
            actual, _ = ops.logits_sample_native(store[:, left : left + 1003], **_to(options, gpu_device))
            assert torch.equal(actual, expected)
    one = (3 * torch.randn(1, 1003, generator=g)).expand(6, 1003)  # one row for all
    _check_sample(one, gpu_device, **options)
    actual, _ = ops.logits_sample_native(one[:1].to(gpu_device).expand(6, 1003), **_to(options, gpu_device))
    assert actual.tolist() == steps.sample(one, **options)[0]


# Rows that several workgroups take.

@pytest.mark.parametrize("dtype", TYPES)
def test_sample_long_rows_of_ties(gpu_device, dtype):
    """More equal logits at the end of what is kept than a list holds, and fewer."""
    g = torch.Generator().manual_seed(19)
    vocab = 20011
    logits = torch.randint(0, 4, (8, vocab), generator=g).to(dtype)
    logits[2] = 0.25  # all equal
    logits[3, ::2], logits[3, 1::2] = -0.0, 0.0
    logits[4:6] = torch.randint(0, 200, (2, vocab), generator=g).to(dtype) / 64
    u = torch.rand(8, generator=g)
    _check_sample(logits, gpu_device, **_options(g, 8, share=0.8))
    _check_sample(logits, gpu_device, uniforms=u, top_k=torch.tensor([1, 4000, 9000, 20010, 1030, 5, 2 ** 40, 1024]))
    _check_sample(logits, gpu_device, uniforms=1 - u / 1000, top_p=torch.tensor([0.1, 0.9, 0.5, 1e-9, 0.2, 0.99, 0.3, 0.7]))
    _check_sample(logits, gpu_device, uniforms=u, top_k=torch.tensor([3000, 300, 9000, 7, 130, 5000, 9, 20000]),
                  top_p=torch.tensor([0.6, 0.9, 0.5, 0.1, 0.2, 0.99, 0.3, 0.7]), min_p=torch.tensor([0.2, 0, 1, 0, 0.5, 0, 0, 0]))


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_long_rows_infinities_and_nan(gpu_device, dtype):
    inf, nan = math.inf, math.nan
    g = torch.Generator().manual_seed(23)
    vocab = 9001
    logits = (2 * torch.randn(9, vocab, generator=g)).to(dtype)
    logits[0, ::2] = -inf
    logits[1, :9000] = -inf
    logits[2] = -inf
    logits[3, 8500], logits[3, 8600] = inf, inf
    logits[4, 40], logits[4, 41] = nan, inf
    logits[5] = torch.finfo(dtype).min
    logits[5, 7:9] = -inf
    logits[6] = torch.finfo(dtype).min
    logits[6, 8999] = torch.finfo(dtype).max
    logits[7, 1:] = -inf
    options = _options(g, 9)
    tokens = _check_sample(logits, gpu_device, **options)
    assert tokens[1:5].tolist() == [9000, 0, 8500, 40] and tokens[6:8].tolist() == [8999, 0]
    _check_sample(logits, gpu_device, uniforms=options["uniforms"], temperature=torch.full((9,), inf))
    _check_sample(logits, gpu_device, uniforms=options["uniforms"], top_k=options["top_k"],
                  temperature=torch.tensor([0.0, 1e-30, 1e-45, -1.0, nan, 1e30, 3e38, 0.01, 1e-38]))


def test_sample_long_rows_strides(gpu_device):
    g = torch.Generator().manual_seed(29)
    logits = 3 * torch.randn(4, 20011, generator=g)
    options = _options(g, 4, share=0.9)
    for dtype in TYPES:
        expected = _check_sample(logits.to(dtype), gpu_device, **options)
        for left in (1, 2, 8):
            store = torch.full((4, 20033), math.nan, device=gpu_device, dtype=dtype)
            store[:, left : left + 20011] = logits.to(dtype)
            assert torch.equal(ops.logits_sample_native(store[:, left : left + 20011], **_to(options, gpu_device))[0], expected)
        # Rows 2^31 elements apart.
        store = torch.empty(3 * 2 ** 31 + 20011, device=gpu_device, dtype=dtype) if dtype != torch.float32 else None
        if store is not None:
            rows = store.as_strided((4, 20011), (2 ** 31, 1))
            rows.copy_(logits.to(dtype))
            assert torch.equal(ops.logits_sample_native(rows, **_to(options, gpu_device))[0], expected)


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 600001), (torch.bfloat16, 1100003)])
def test_sample_large_vocabularies(gpu_device, dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    logits = (2 * torch.randn(1, vocab, generator=g)).to(dtype)
    u = torch.rand(1, generator=g)
    _check_sample(logits, gpu_device, uniforms=u)
    _check_sample(logits, gpu_device, uniforms=u, top_k=torch.tensor([50]), top_p=torch.tensor([0.7]), min_p=torch.tensor([0.01]))


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_the_largest_vocabulary(gpu_device, dtype):
    """Sixteen million tokens, a few of which are possible, the first and the last among them."""
    vocab = 1 << 24
    places = torch.tensor([0, 1, 511, 512, 70000, 8388607, 8388608, vocab - 2, vocab - 1])
    few = torch.tensor([[1.0, 0.5, 2.0, 0.0, 1.0, 1.5, -1.0, 0.25, 1.0]])
    row = torch.full((1, vocab), -math.inf, device=gpu_device, dtype=dtype)
    row[0, places.to(gpu_device)] = few[0].to(gpu_device).to(dtype)
    for u in (0.0, 0.1, 0.3, 0.5, 0.7, 0.8, 0.9, 0.95, 1 - 2.0 ** -24):
        for options in ({}, {"top_k": torch.tensor([4])}, {"top_p": torch.tensor([0.9]), "top_k": torch.tensor([8])},
                        {"min_p": torch.tensor([0.3])}):
            options = {"uniforms": torch.tensor([u]), **options}
            token, _ = ops.logits_sample_native(row, **_to(options, gpu_device))
            assert int(token) == int(places[steps.sample(few, **options)[0][0]])


# --------------------------------------------------------------------------- together

class _Server:
    """A served loop of one layer, its tensors on the GPU and the oracle's on the host."""

    def __init__(self, device, dtype, seed, slots=6, columns=12, page_size=16, heads=6, kv_heads=2, dim=64, vocab=300, pages=60):
        g = torch.Generator().manual_seed(seed)
        self.g, self.device, self.dtype, self.shape = g, device, dtype, (heads, kv_heads, dim)
        self.page_size, self.slots = page_size, slots
        self.books = ref.Pages(1, pages, kv_heads, page_size, dim, slots, columns, dtype, seed)
        self.key, self.value = self.books.key[0].to(device), self.books.value[0].to(device)
        self.table = torch.full((slots, columns), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(slots, dtype=torch.int64, device=device)
        self.refcounts = torch.zeros(pages, dtype=torch.int32, device=device)
        self.embedding = torch.randn(vocab, heads + 2 * kv_heads, dim, generator=g).to(dtype)
        self.head = torch.randn(heads * dim, vocab, generator=g).to(dtype)

    def step(self, tokens, slots, counts, ids, uniforms, options):
        """On the GPU; returns what the oracle computes as well."""
        heads, kv_heads, dim = self.shape
        positions, _ = ops.paged_cache_reserve_native(self.table, self.lengths, self.refcounts, self.page_size, slots, counts)
        offsets, request, position, rows = ops.paged_step_layout_native(self.table, slots, positions, counts, self.page_size, tokens)
        packed = self.embedding.to(self.device)[ids]
        ops.paged_cache_write_rows_native(packed[:, heads : heads + kv_heads], packed[:, heads + kv_heads :], self.key, self.value, rows)
        out = ops.paged_chunk_attention_native(packed[:, :heads], self.key, self.value, self.table, self.lengths, offsets, dim ** -0.5,
                                               0, 0, slots, positions)
        last = (offsets[1:] - 1).clamp(min=0)
        logits = out[last].flatten(1) @ self.head.to(self.device)
        token, share = ops.logits_sample_native(logits, uniforms, **options)
        return positions, offsets, request, position, rows, out, logits, token, share

    def expected(self, tokens, slots, counts, ids, got):
        heads, kv_heads, dim = self.shape
        positions, _ = self.books.reserve(slots.tolist(), counts.tolist())
        table = torch.tensor(self.books.table, dtype=torch.int32)
        assert got[0].tolist() == positions and self.table.cpu().equal(table)
        places = steps.step_layout(table, slots, torch.tensor(positions), counts, self.page_size, tokens)
        assert [t.tolist() for t in got[1:5]] == list(places)
        packed = self.embedding[ids]
        steps.write_rows(packed[:, heads : heads + kv_heads], packed[:, heads + kv_heads :], self.books.key[0], self.books.value[0],
                         torch.tensor(places[3]))
        assert torch.equal(self.key.cpu(), self.books.key[0]) and torch.equal(self.value.cpu(), self.books.value[0])
        case = {"query": packed[:, :heads], "key_pages": self.books.key[0], "value_pages": self.books.value[0], "page_table": table,
                "lengths": torch.tensor(self.books.lengths), "offsets": torch.tensor(places[0]), "scale": dim ** -0.5}
        out = steps.chunk_attention(**case, slots=slots, positions=torch.tensor(positions))
        _close(got[5], out, _bound(case, out))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_served_loop_of_mixed_steps(gpu_device, dtype):
    """Chunks of prompts next to tokens, a refused request, sequences that end and others that take their slots."""
    server = _Server(gpu_device, dtype, 41)
    rng = random.Random(43)
    g = torch.Generator().manual_seed(47)
    for turn in range(10):
        count = rng.randint(1, 6)
        slots = torch.tensor(rng.sample(range(7), count))  # slot 6 is outside the table
        counts = torch.tensor([rng.choice((1, 1, 5, 33, 60)) for _ in range(count)])
        tokens = 220
        ids = torch.randint(0, 300, (tokens,), generator=g)
        uniforms, options = torch.rand(count, generator=g), _options(g, count)
        options.pop("uniforms")
        got = server.step(tokens, slots.to(gpu_device), counts.to(gpu_device), ids.to(gpu_device), uniforms.to(gpu_device),
                          _to(options, gpu_device))
        server.expected(tokens, slots, counts, ids, got)
        assert got[7].tolist() == steps.sample(got[6].cpu(), uniforms, **options)[0]
        if turn % 3 == 2:
            gone = rng.sample(range(6), 2)
            ops.paged_cache_free_native(server.table, server.lengths, server.refcounts, torch.tensor(gone, device=gpu_device))
            server.books.free(gone)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_captured_step_is_replayed(gpu_device, dtype):
    """One graph for steps of every composition up to its size, between eager steps of another server."""
    server, eager = (_Server(gpu_device, dtype, 53, columns=80, pages=400) for _ in range(2))
    g = torch.Generator().manual_seed(59)
    tokens, requests = 150, 5
    slots, counts = torch.arange(requests, device=gpu_device), torch.ones(requests, dtype=torch.int64, device=gpu_device)
    ids, uniforms = torch.zeros(tokens, dtype=torch.int64, device=gpu_device), torch.zeros(requests, device=gpu_device)
    options = _to(_options(g, requests), gpu_device)
    options.pop("uniforms")
    for s in (server, eager):  # long contexts, so that tiles are cut
        s.embedding, s.head = s.embedding.to(gpu_device), s.head.to(gpu_device)
        s.step(1300, slots[:2], torch.tensor([1000, 300], device=gpu_device), torch.randint(0, 300, (1300,), generator=torch.Generator().manual_seed(1)).to(gpu_device),
               uniforms[:2], {})
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    before = [t.clone() for t in (server.key, server.value, server.table, server.lengths, server.refcounts)]
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        server.step(tokens, slots, counts, ids, uniforms, options)
    torch.cuda.current_stream().wait_stream(stream)
    for t, b in zip((server.key, server.value, server.table, server.lengths, server.refcounts), before):
        t.copy_(b)
    with torch.cuda.graph(graph):
        got = server.step(tokens, slots, counts, ids, uniforms, options)
    for turn in range(6):
        slots.copy_(torch.randperm(6, generator=g)[:requests])
        counts.copy_(torch.tensor([1, 1, 20, 0, 90])[torch.randperm(5, generator=g)])
        ids.copy_(torch.randint(0, 300, (tokens,), generator=g))
        uniforms.copy_(torch.rand(requests, generator=g))
        graph.replay()
        expected = eager.step(tokens, slots, counts, ids, uniforms, options)
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(got, expected)), turn
        assert torch.equal(server.key, eager.key) and torch.equal(server.table, eager.table)


def test_steps_on_another_stream(gpu_device):
    case = _to(_chunk_case(61, torch.bfloat16, 4, 2, 64, 16, [(40, 500), (1, 3000)]), gpu_device)
    logits = 3 * torch.randn(4, 30000, device=gpu_device)
    u = torch.rand(4, device=gpu_device)
    expected = ops.paged_chunk_attention_native(**case), *ops.logits_sample_native(logits, u)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(1_000_000)
        moved = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in case.items()}
        later = logits.clone()
        actual = ops.paged_chunk_attention_native(**moved), *ops.logits_sample_native(later, u)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, e) for a, e in zip(actual, expected))


def test_two_streams_at_once(gpu_device):
    """Calls whose tiles are cut and joined, and rows of several workgroups, side by side on two streams."""
    cases = [_to(_chunk_case(91 + i, dtype, 4, 2, 64, 16, [(40, 5000), (1, 9000), (300 * i, 20)]), gpu_device)
             for i, dtype in enumerate((torch.bfloat16, torch.float32))]
    logits = [3 * torch.randn(4, 30000 + 7 * i, device=gpu_device) for i in range(2)]
    u = torch.rand(4, device=gpu_device)
    k = torch.tensor([0, 5, 100, 3000], device=gpu_device)

    def call(i):
        return ops.paged_chunk_attention_native(**cases[i]), *ops.logits_sample_native(logits[i], u, top_k=k)

    expected = [call(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, e) for i in range(2) for one in got[i] for a, e in zip(one, expected[i]))
