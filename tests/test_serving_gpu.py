"""GPU parity of the serving operators against plain float64 forms (``oracle/serving.py``) and Python page books.

Tolerances of the attention operators are computed from the inputs (``oracle.serving.attention_bound``); everything that
moves values or counts is exact, and processed logits are the float32 operations of the definition rounded once.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from flux_amd import ops
from oracle import serving as ref

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _close(actual, expected, bound):
    error = (actual.cpu().double() - expected).abs()
    beyond = float((error - bound).nan_to_num(nan=math.inf).max())
    assert beyond <= 0, f"off by {beyond:.3g} beyond the bound, at most {float(error.max()):.3g}"


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g).to(dtype)


def _paged_case(seed, dtype, heads, kv_heads, dim, page_size, lengths, spare=3, scale=None):
    """CPU tensors of a batch whose pages lie scattered in the pool."""
    g = torch.Generator().manual_seed(seed)
    columns = max(1, -(-max(max(lengths), 1) // page_size))
    needed = [-(-n // page_size) for n in lengths]
    pages = sum(needed) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lengths), columns), -1, dtype=torch.int32)
    for b, count in enumerate(needed):
        for c in range(count):
            table[b, c] = order.pop()
    return {"query": _randn(g, (len(lengths), heads, 1, dim), dtype),
            "key_pages": _randn(g, (pages, kv_heads, page_size, dim), dtype),
            "value_pages": _randn(g, (pages, kv_heads, page_size, dim), dtype),
            "page_table": table, "lengths": torch.tensor(lengths), "scale": scale or dim ** -0.5}


def _to(case, device):
    return {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in case.items()}


def _check_paged(case, device, actual=None, **options):
    expected = ref.paged_decode(**case, **{k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in options.items()})
    if actual is None:
        options = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in options.items()}
        actual = ops.paged_decode_attention_native(**_to(case, device), **options)
    assert actual.dtype == case["query"].dtype and actual.is_contiguous() and actual.shape == expected.shape
    terms = int(min(case["lengths"].max(), case["page_table"].shape[1] * case["key_pages"].shape[2]))
    _close(actual, expected, ref.attention_bound(case["query"], case["key_pages"].nan_to_num(), case["value_pages"].nan_to_num(),
                                                 case["scale"], max(terms, 1), case["query"].dtype, expected))
    return actual


# --------------------------------------------------------------------------- paged decode

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,page_size", [(64, 16), (128, 64), (256, 16), (80, 48), (72, 7), (40, 1), (100, 5), (5, 3),
                                           (1, 4), (192, 100), (33, 16)])
def test_paged_decode_heads_and_pages(gpu_device, dtype, dim, page_size):
    lengths = [1, 0, 15, 16, 17, 31, 33, 64, 127, 200, 301]
    for heads, kv_heads in ((9, 3), (4, 4), (20, 1)):
        case = _paged_case(dim + page_size, dtype, heads, kv_heads, dim, page_size, lengths)
        out = _check_paged(case, gpu_device)
        assert not out[1].any()


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 9), (1, 0), (1, 1), (16, 0), (31, 4), (32, 33), (100, 1), (150, 64),
                                          (1000, 5), (1 << 24, 1 << 24)])
@pytest.mark.parametrize("dtype,dim,page_size", [(torch.float32, 64, 16), (torch.bfloat16, 128, 24),
                                                 (torch.float16, 256, 33)])
def test_paged_decode_windows(gpu_device, dtype, dim, page_size, window, sinks):
    case = _paged_case(7, dtype, 6, 2, dim, page_size, [1, 0, 2, 16, 32, 33, 101, 130, 257, 400])
    _check_paged(case, gpu_device, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
def test_paged_decode_long_and_large_batches(gpu_device, dtype):
    """Sequences that are cut over many workgroups next to short ones, and more sequences than one round's threads."""
    _check_paged(_paged_case(1, dtype, 3, 1, 64, 16, [9000, 3, 700, 0, 5000]), gpu_device)
    rng = random.Random(2)
    lengths = [rng.choice((0, 1, 5, 40, 90)) for _ in range(601)]
    lengths[0] = lengths[300] = 0
    _check_paged(_paged_case(3, dtype, 2, 2, 32, 8, lengths), gpu_device)


# Inputs whose results tell every key: the score of key j is -(j // 16 % 8) times the head's factor, so that with a scale of
# ln 2 its weight is a power of two, and its value is 1 in the dim j // 16 % D and 0 in all others.

def _telling_keys(count, dim, dtype):
    tile = torch.arange(count) // 16
    key, value = torch.zeros(count, dim, dtype=dtype), torch.zeros(count, dim, dtype=dtype)
    key[:, 0] = -(tile % 8).to(dtype)
    value[torch.arange(count), tile % dim] = 1
    return key, value


def _telling_query(shape, dtype):
    query = torch.zeros(shape, dtype=dtype)
    query[..., 0] = (1 + torch.arange(shape[1]) % 2).to(dtype).view(1, -1, 1)
    return query


def _telling_bound(expected, dtype, additions):
    """Relative, as all terms are positive.  The exponent of a weight, at most 32 below the running maximum's, is off by 3
    2^-24 of itself, together with the steps that the maximum takes: 32 * 3 * 2^-24 ln 2 < 2^-17 of the weight, and 2^-22 for
    each of at most 20 exponentials, < 2^-17.  What a power of two that is off by this leaves in 16 bits is below 2^-17 again.
    ``additions``, one after the other, are off by 2^-24 each, in the sums of the weights and of the values; the quotient by
    2^-23; and the result is rounded once."""
    relative = 2.0 ** -15 + additions * 2.0 ** -23 + torch.finfo(dtype).eps / 2
    return relative * expected + torch.finfo(dtype).tiny


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 1, 64), (20, 1, 128), (4, 2, 80), (2, 1, 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2000, 40)])
def test_paged_decode_loses_no_key_where_sequences_are_cut(gpu_device, dtype, heads, kv_heads, dim, window, sinks):
    lengths, page_size = [9000, 3, 700, 0, 5000, 16, 1999], 48
    case = _paged_case(67, dtype, heads, kv_heads, dim, page_size, lengths, scale=math.log(2))
    case["query"] = _telling_query(case["query"].shape, dtype)
    for b, n in enumerate(lengths):
        key, value = _telling_keys(-(-n // page_size) * page_size, dim, dtype)
        for c in range(-(-n // page_size)):
            page = int(case["page_table"][b, c])
            case["key_pages"][page] = key[c * page_size : (c + 1) * page_size]
            case["value_pages"][page] = value[c * page_size : (c + 1) * page_size]
    expected = ref.paged_decode(**case, window=window, sinks=sinks)
    # 2 tiles of a wave and as many additions a key as a lane makes, four waves, 71 parts.
    bound = _telling_bound(expected, dtype, 128)
    _close(ops.paged_decode_attention_native(**_to(case, gpu_device), window=window, sinks=sinks), expected, bound)
    # The bound tells a lost tile of 16 keys, wherever it lies.
    for b, n in enumerate(lengths):
        key, value = _telling_keys(n, dim, dtype)
        for first in {0, n // 3 // 16 * 16, (n - 1) // 16 * 16} if n > 16 else ():
            seen = [j for j in ref.visible_keys(n - 1, n, window, sinks)]
            kept = [j for j in seen if not first <= j < first + 16]
            if len(kept) < len(seen):
                lost = ref.attend(case["query"][b, 0, 0], key[kept], value[kept], case["scale"])
                assert bool(((lost - expected[b, 0, 0]).abs() > bound[b, 0, 0]).any())


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.float32, 128), (torch.float16, 64), (torch.bfloat16, 128)])
def test_paged_decode_joins_more_parts_than_it_keeps_shares_of(gpu_device, dtype, dim):
    """One sequence in hundreds of parts: a far larger key behind the 128th part, parts whose keys are all left out (no page, or
    a score of -inf) before and behind it."""
    n, page_size = 33000, 16
    case = _paged_case(71, dtype, 3, 1, dim, page_size, [n], scale=math.log(2))
    case["query"] = _telling_query(case["query"].shape, dtype)
    key, value = _telling_keys(case["page_table"].shape[1] * page_size, dim, dtype)
    key[30000, 0] = 8
    for gone in (6400, 27520):  # 320 keys hold a whole part of 128 or 80, wherever it starts
        key[gone : gone + 320, 0] = -math.inf
    table = case["page_table"][0].long()
    case["key_pages"][table] = key.view(-1, 1, page_size, dim)
    case["value_pages"][table] = value.view(-1, 1, page_size, dim)
    for gone in (3200, 25600):
        case["page_table"][0, gone // page_size : (gone + 320) // page_size] = -1
    device = _to(case, gpu_device)
    needed = ops.paged_decode_workspace_bytes(device["query"], device["key_pages"], device["page_table"]) // 4
    output, workspace = torch.empty_like(device["query"]), torch.empty(needed, device=gpu_device)
    ops.paged_decode_attention_native_out(*device.values(), 0, 0, None, output, workspace)
    first, parts = workspace[-2:].view(torch.int32).tolist()
    assert first == 0 and parts > 200
    expected = ref.paged_decode(**case)
    assert bool(expected.isfinite().all())
    bound = _telling_bound(expected, dtype, 64 + parts)
    _close(output, expected, bound)
    # The bound tells a part behind the 128th, or its share taken for 1.
    weights = torch.exp2(key[:, 0].double())
    weights[[*range(3200, 3520), *range(25600, 25920)]] = 0
    weights[n:] = 0
    for changed in (0.0, 2.0 ** 8):
        other = weights.clone()
        other[26880:27008] *= changed
        moved = (other @ value.double()) / other.sum()
        assert bool(((moved - expected[0, 0, 0]).abs() > bound[0, 0, 0]).any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 1, 64), (6, 2, 128), (2, 1, 80), (2, 1, 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (500, 21), (37, 0)])
def test_window_attention_loses_no_key(gpu_device, dtype, heads, kv_heads, dim, window, sinks):
    """A chunk, a prompt and a token at the end of long keys."""
    for queries, keys in ((40, 2000), (330, 330), (1, 9000)):
        key, value = _telling_keys(keys, dim, dtype)
        case = {"query": _telling_query((1, heads, queries, dim), dtype), "key": key.expand(1, kv_heads, keys, dim),
                "value": value.expand(1, kv_heads, keys, dim), "scale": math.log(2)}
        expected = ref.window_attention(**case, window=window, sinks=sinks)
        bound = _telling_bound(expected, dtype, keys // 4)  # two lanes share a row and add its weights in pairs
        _close(ops.window_attention_native(**_to(case, gpu_device), window=window, sinks=sinks), expected, bound)
        seen = ref.visible_keys(keys - 1, keys, window, sinks)
        for first in (seen[0], seen[len(seen) // 2], seen[-1] - 15):
            kept = [j for j in seen if not first <= j < first + 16]
            lost = ref.attend(case["query"][0, 0, -1], key[kept], value[kept], case["scale"])
            assert bool(((lost - expected[0, 0, -1]).abs() > bound[0, 0, -1]).any())


def test_paged_decode_one_sequence_at_every_length(gpu_device):
    case = _paged_case(11, torch.float32, 9, 3, 64, 16, [300])
    device = _to(case, gpu_device)
    for n in [*range(0, 70), 127, 128, 129, 255, 256, 257, 299, 300]:
        case["lengths"] = torch.tensor([n])
        device["lengths"] = case["lengths"].to(gpu_device)
        _check_paged(case, gpu_device, ops.paged_decode_attention_native(**device))


def test_paged_decode_slots_lengths_and_bad_pages(gpu_device):
    case = _paged_case(13, torch.float32, 6, 2, 64, 16, [50, 200, 33, 120])
    # Rows in another order, twice, and outside the table; lengths beyond the columns and negative ones.
    case["query"] = torch.randn(7, 6, 1, 64, generator=torch.Generator().manual_seed(1))
    slots = torch.tensor([2, 0, 4, -1, 1, 1, 3])
    out = _check_paged(case, gpu_device, slots=slots)
    assert not out[2].any() and not out[3].any()
    case["lengths"] = torch.tensor([1 << 40, -5, 33, 120])
    _check_paged(case, gpu_device, slots=slots)
    # Entries outside the pool are left out: the sequence attends over the others.
    case["lengths"] = torch.tensor([50, 200, 33, 120])
    case["page_table"][0, 1] = -1
    case["page_table"][1, 3] = case["key_pages"].shape[0]
    case["page_table"][1, 4] = 2 ** 31 - 1
    case["page_table"][2] = -7
    out = _check_paged(case, gpu_device, slots=slots)
    assert not out[0].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_paged_decode_strides_and_alignment(gpu_device, dtype):
    case = _paged_case(17, dtype, 6, 2, 64, 16, [50, 200, 33, 120])
    expected = ops.paged_decode_attention_native(**_to(case, gpu_device))
    device = _to(case, gpu_device)
    # [P, page, heads, D] pages, a table inside a wider one, a query inside a packed projection, another dim stride.
    moved = dict(device)
    for name in ("key_pages", "value_pages"):
        moved[name] = device[name].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((4, 40), 99, dtype=torch.int32, device=gpu_device)
    wide[:, 3:3 + device["page_table"].shape[1]] = device["page_table"]
    moved["page_table"] = wide[:, 3:3 + device["page_table"].shape[1]]
    packed = torch.randn(4, 3, 6, 64, device=gpu_device).to(dtype)
    packed[:, 1] = device["query"][:, :, 0]
    moved["query"] = packed[:, 1].unsqueeze(2)
    assert torch.equal(ops.paged_decode_attention_native(**moved), expected)
    moved["query"] = device["query"].transpose(1, 3).contiguous().transpose(1, 3)
    assert torch.equal(ops.paged_decode_attention_native(**moved), expected)
    # Rows that start at no 16 bytes.
    for name in ("key_pages", "value_pages"):
        shape = device[name].shape
        store = torch.randn(shape[0], shape[1], shape[2], 67, device=gpu_device).to(dtype)
        store[..., 1:65] = device[name]
        moved[name] = store[..., 1:65]
    torch.testing.assert_close(ops.paged_decode_attention_native(**moved), expected, rtol=0, atol=0)


def test_paged_decode_ignores_what_lies_behind(gpu_device):
    """NaN and infinity in rows behind the length, before the window and on other pages."""
    case = _paged_case(19, torch.bfloat16, 8, 2, 128, 16, [50, 200, 33, 120])
    window, sinks = 20, 3
    clean = ops.paged_decode_attention_native(**_to(case, gpu_device), window=window, sinks=sinks)
    seen = torch.zeros(case["key_pages"].shape[0], 16, dtype=torch.bool)
    for b, n in enumerate(case["lengths"].tolist()):
        for j in ref.visible_keys(n - 1, n, window, sinks):
            seen[int(case["page_table"][b, j // 16]), j % 16] = True
    for bad in (math.nan, math.inf, -math.inf):
        for name in ("key_pages", "value_pages"):
            case[name] = torch.where(seen[:, None, :, None], case[name], torch.tensor(bad, dtype=torch.bfloat16))
        assert torch.equal(ops.paged_decode_attention_native(**_to(case, gpu_device), window=window, sinks=sinks), clean)


def test_paged_decode_nan_and_large_scores(gpu_device):
    case = _paged_case(23, torch.float32, 2, 1, 64, 16, [40, 40])
    page = int(case["page_table"][1, 1])
    case["value_pages"][page, 0, 3, 7] = math.nan
    out = ops.paged_decode_attention_native(**_to(case, gpu_device)).cpu()
    assert out[0].isfinite().all() and out[1, :, 0, 7].isnan().all()
    assert out[1, :, 0].isnan().sum() == 2
    case["key_pages"][page, 0, 3] = math.nan
    assert ops.paged_decode_attention_native(**_to(case, gpu_device)).cpu()[1].isnan().all()
    # Scores around 1e38 leave the largest one alone.
    case = _paged_case(29, torch.float32, 1, 1, 64, 16, [70])
    case["query"] = torch.full_like(case["query"], 1e18)
    case["key_pages"] = case["key_pages"].abs() * 1e18
    case["scale"] = 1.0
    out = ops.paged_decode_attention_native(**_to(case, gpu_device)).cpu().double()
    expected = ref.paged_decode(**case)
    torch.testing.assert_close(out, expected, rtol=1e-6, atol=0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 80, 100, 5, 136, 129])
def test_a_key_of_infinities_has_no_weight(gpu_device, dtype, dim):
    """A key whose score is -inf is as good as masked, also where the head does not fill the registers' dims."""
    case = _paged_case(37, dtype, 4, 2, dim, 16, [50, 33])
    case["query"][..., 0] = case["query"][..., 0].abs() + 0.5
    finite = {**case, "key_pages": case["key_pages"].clone()}
    for b, position in ((0, 3), (0, 49), (1, 20)):
        case["key_pages"][int(case["page_table"][b, position // 16]), :, position % 16, 0] = -math.inf
    expected = ref.paged_decode(**case)
    assert bool(expected.isfinite().all())
    bound = ref.attention_bound(finite["query"], finite["key_pages"], finite["value_pages"], finite["scale"], 50, dtype, expected)
    _close(ops.paged_decode_attention_native(**_to(case, gpu_device)), expected, bound)

    case = _window_case(41, dtype, 1, 4, 2, dim, 40, 40)
    case["query"][..., 0] = case["query"][..., 0].abs() + 0.5
    finite = {**case, "key": case["key"].clone()}
    case["key"][:, :, [5, 22], 0] = -math.inf
    expected = ref.window_attention(**case, window=0)
    assert bool(expected.isfinite().all())
    bound = ref.attention_bound(finite["query"], finite["key"], finite["value"], finite["scale"], 40, dtype, expected, True)
    _close(ops.window_attention_native(**_to(case, gpu_device), window=0), expected, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page_size", [(9, 3, 64, 16), (20, 1, 128, 24), (4, 2, 80, 16), (6, 2, 5, 7), (2, 1, 256, 33),
                                                          (3, 3, 100, 48)])
def test_infinite_values_stay_infinite(gpu_device, dtype, heads, kv_heads, dim, page_size):
    """A visible infinity times a weight above zero is an infinity of its sign; two of both signs are NaN.  Also behind small
    weights, in sequences that are cut over workgroups, and next to NaN."""
    case = _paged_case(59, dtype, heads, kv_heads, dim, page_size, [40, 2500, 2500, 33])
    finite = {**case, "value_pages": case["value_pages"].clone()}

    def place(b, position):
        return int(case["page_table"][b, position // page_size]), slice(None), position % page_size

    for b, position, d, value in ((0, 5, 0, math.inf), (0, 39, 1, -math.inf), (1, 5, 2, math.inf), (1, 1700, 2, math.inf),
                                  (1, 2499, 3, math.inf), (1, 20, 3, -math.inf), (2, 700, 4, math.nan), (2, 701, 4, math.inf)):
        case["value_pages"][place(b, position)][..., d] = value
    # Its score lies 40 below the others' middle: a weight that 16 bits do not hold next to the largest.
    low = place(0, 5)
    for h in range(kv_heads):
        q = case["query"][0, h * (heads // kv_heads), 0].double()
        case["key_pages"][low[0], h, low[2]] = (-40 / case["scale"] * q / q.dot(q).clamp(min=0.1)).to(dtype)
    finite["key_pages"] = case["key_pages"]
    expected = ref.paged_decode(**case)
    assert bool(expected[0, ..., 0].isinf().any()) and bool(expected[1, ..., 3].isnan().all()) and bool(expected[3].isfinite().all())
    bound = ref.attention_bound(finite["query"], finite["key_pages"], finite["value_pages"], case["scale"], 2500, dtype, expected)
    out = ops.paged_decode_attention_native(**_to(case, gpu_device)).cpu()
    for sign in (math.inf, -math.inf):
        assert torch.equal(out == sign, expected == sign)
    assert torch.equal(out.isnan(), expected.isnan())
    kept = expected.isfinite()
    _close(out[kept], expected[kept], bound[kept])

    # One run of keys per sequence, one token and several.
    for queries in (1, 3):
        case = _window_case(61, dtype, 2, heads, kv_heads, dim, queries, 300)
        case["value"][0, :, 7, 0], case["value"][0, :, 250, 1], case["value"][1, :, 299, 2] = math.inf, -math.inf, math.inf
        expected = ref.window_attention(**case, window=100, sinks=8)
        out = ops.window_attention_native(**_to(case, gpu_device), window=100, sinks=8).cpu()
        for sign in (math.inf, -math.inf):
            assert torch.equal(out == sign, expected == sign)
        assert torch.equal(out.isnan(), expected.isnan()) and not bool(out.isnan().any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 80])
def test_scores_that_are_all_minus_infinity_give_zeros(gpu_device, dtype, dim):
    case = _to(_window_case(43, dtype, 1, 4, 2, dim, 40, 40), gpu_device)
    case["query"][..., 0] = case["query"][..., 0].abs() + 0.5
    case["key"][:, :, :20, 0] = -math.inf
    out = ops.window_attention_native(**case, window=8, sinks=2)
    assert not bool(out[:, :, :20].any()) and bool(out[:, :, 20:].isfinite().all()) and bool(out[:, :, 20:].any())
    for n in (1, 20, 21):
        one = ops.window_attention_native(**{**case, "query": case["query"][:, :, n - 1 : n]}, window=8, sinks=2,
                                          lengths=torch.tensor([n], device=gpu_device))
        assert bool(one.isfinite().all()) and bool(one.any()) == (n > 20)


def test_paged_decode_many_small_weights_in_float16(gpu_device):
    """One key far above 8000 others whose weights are below float16's smallest step together weigh a fifth."""
    n = 8192
    case = _paged_case(31, torch.float16, 1, 1, 64, 64, [n], scale=1.0)
    case["query"] = torch.zeros(1, 1, 1, 64, dtype=torch.float16)
    case["query"][..., 0] = 1.0
    case["key_pages"] = torch.zeros_like(case["key_pages"])
    case["key_pages"][..., 0] = -10.5
    first = int(case["page_table"][0, 0])
    case["key_pages"][first, 0, 0, 0] = 0.0
    case["value_pages"] = torch.ones_like(case["value_pages"])
    case["value_pages"][first, 0, 0] = -1.0
    out = ops.paged_decode_attention_native(**_to(case, gpu_device)).cpu().double()
    rest = (n - 1) * math.exp(-10.5)
    expected = (rest - 1) / (rest + 1)
    assert abs(float(out[0, 0, 0, 5]) - expected) <= 2.0 ** -11 * abs(expected) + 1e-5


def test_paged_decode_out_streams_and_reuse(gpu_device):
    case = _paged_case(37, torch.float32, 9, 3, 64, 16, [900, 30, 2000])
    device = _to(case, gpu_device)
    expected = _check_paged(case, gpu_device)
    needed = ops.paged_decode_workspace_bytes(device["query"], device["key_pages"], device["page_table"])
    output = torch.full_like(device["query"], 7.0)
    workspace = torch.full((needed // 4 + 64,), math.nan, device=gpu_device)
    call = lambda o, w: ops.paged_decode_attention_native_out(*device.values(), 0, 0, None, o, w)  # noqa: E731
    assert call(output, workspace) is output
    assert torch.equal(output, expected) and workspace[needed // 4:].isnan().all()
    with pytest.raises(RuntimeError, match="workspace is too small"):
        call(output, workspace[: needed // 4 - 1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        others = [ops.paged_decode_attention_native(**device) for _ in range(3)]
    here = [ops.paged_decode_attention_native(**device) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, expected) for t in others + here)


def test_paged_decode_matches_the_one_sequence_operator(gpu_device):
    g = torch.Generator().manual_seed(41)
    cache = torch.randn(2, 1, 3, 1024, 64, generator=g).to(gpu_device)
    query = torch.randn(1, 9, 1, 64, generator=g).to(gpu_device)
    length = torch.tensor(777, device=gpu_device)
    one = ops.gqa_decode_attention_native(query, cache[0], cache[1], None, 0.125, length)
    pages = [c[0].view(3, 64, 16, 64).transpose(0, 1) for c in cache]
    table = torch.arange(64, dtype=torch.int32, device=gpu_device)[None]
    paged = ops.paged_decode_attention_native(query, *pages, table, length[None], 0.125)
    whole = ops.window_attention_native(query, cache[0], cache[1], 0.125, 0, 0, length[None])
    torch.testing.assert_close(paged, one, rtol=2e-5, atol=1e-6)
    torch.testing.assert_close(whole, one, rtol=2e-5, atol=1e-6)


# --------------------------------------------------------------------------- window attention

def _window_case(seed, dtype, batch, heads, kv_heads, dim, queries, keys):
    g = torch.Generator().manual_seed(seed)
    return {"query": _randn(g, (batch, heads, queries, dim), dtype), "key": _randn(g, (batch, kv_heads, keys, dim), dtype),
            "value": _randn(g, (batch, kv_heads, keys, dim), dtype), "scale": dim ** -0.5}


def _check_window(case, device, window, sinks=0, lengths=None, starts=None):
    lengths = None if lengths is None else torch.tensor(lengths)
    starts = None if starts is None else torch.tensor(starts)
    expected = ref.window_attention(**case, window=window, sinks=sinks, lengths=lengths, starts=starts)
    actual = ops.window_attention_native(**_to(case, device), window=window, sinks=sinks,
                                         lengths=None if lengths is None else lengths.to(device),
                                         starts=None if starts is None else starts.to(device))
    assert actual.dtype == case["query"].dtype and actual.is_contiguous()
    terms = case["key"].shape[2] if window == 0 else min(case["key"].shape[2], window + sinks)
    _close(actual, expected, ref.attention_bound(case["query"], case["key"], case["value"], case["scale"], max(terms, 1),
                                                 case["query"].dtype, expected, case["query"].shape[2] > 1))
    return actual


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 9, 3), (128, 8, 2), (256, 2, 1), (80, 3, 3), (72, 5, 1), (40, 20, 1),
                                                (100, 2, 2), (5, 4, 2), (1, 1, 1), (192, 2, 1)])
def test_window_heads(gpu_device, dtype, dim, heads, kv_heads):
    for queries, keys in ((2, 2), (35, 35), (17, 90), (1, 70)):
        _check_window(_window_case(dim, dtype, 2, heads, kv_heads, dim, queries, keys), gpu_device, 20, 3)


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.float16, 64), (torch.bfloat16, 128), (torch.float32, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 3), (1, 0), (1, 1), (2, 0), (16, 0), (31, 4), (33, 40), (64, 1),
                                          (150, 0), (1 << 24, 1 << 24)])
def test_window_sizes(gpu_device, dtype, dim, window, sinks):
    _check_window(_window_case(3, dtype, 1, 3, 1, dim, 150, 150), gpu_device, window, sinks)
    _check_window(_window_case(5, dtype, 1, 2, 2, dim, 40, 170), gpu_device, window, sinks)
    _check_window(_window_case(6, dtype, 1, 2, 2, dim, 1, 170), gpu_device, window, sinks)


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.float16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
def test_window_scales(gpu_device, dtype, dim, scale):
    for queries in (60, 1):
        case = {**_window_case(8, dtype, 1, 3, 1, dim, queries, 90), "scale": scale}
        _check_window(case, gpu_device, 20, 2)
        _check_window(case, gpu_device, 0, 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("below", [20, 24, 30, 31, 33, 35])
def test_window_many_small_weights_over_a_long_run(gpu_device, dtype, below):
    """One key whose value is 0 far above n = 2^22 others, each 2^-below of it: what they add up to must not be lost.

    The scale is ln 2, so that a weight is 2^-below (1 + d) with |d| <= below 3 2^-24 ln 2 + 2^-22 < 2^-17, which both types
    round to 2^-below itself; its products with powers of two add up without rounding (at most 2^22 multiples of the
    smallest).  The sum of the weights lies between that of the large one alone, in whose lane a float32 sum may lose the
    others, and that of all, both within 2^-17; the result is rounded once, by half a step.
    """
    n, dim = 1 << 22, 8
    query, key = torch.zeros(1, 1, 2, dim, dtype=dtype), torch.full((1, 1, n, dim), 0.0, dtype=dtype)
    query[..., 0] = 1
    key[..., 0] = -below
    key[0, 0, 0, 0] = 0
    each = torch.tensor([1, -2, 0.25, 4, -0.5, 1, 2, 0])
    value = each.to(dtype).repeat(1, 1, n, 1)
    value[0, 0, 0] = 0
    out = ops.window_attention_native(query.to(gpu_device), key.to(gpu_device), value.to(gpu_device), math.log(2), 0).cpu().double()
    for row, count in ((0, n - 2), (1, n - 1)):
        rest = count * 2.0 ** -below
        slack = torch.finfo(dtype).eps / 2 + 2.0 ** -16
        size = out[0, 0, row] / each.double().where(each != 0, torch.tensor(1.0, dtype=torch.float64))
        assert float(size[7]) == 0
        assert bool((size[:7] >= rest / (1 + rest) * (1 - slack)).all()) and bool((size[:7] <= rest * (1 + slack)).all()), (size, rest)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 40])
def test_window_scale_of_zero_makes_infinite_scores_nan(gpu_device, dtype, dim):
    """0 * inf is NaN, for one query as for many; rows that do not see the key are means of their values."""
    case = {**_window_case(47, dtype, 1, 3, 1, dim, 40, 40), "scale": 0.0}
    case["query"][..., 0] = case["query"][..., 0].abs() + 0.5
    finite = {**case, "key": case["key"].clone()}
    case["key"][0, 0, 25, 0] = -math.inf
    expected = ref.window_attention(**case, window=10)
    lost = expected.isnan().all(-1)[0, 0]
    assert lost.nonzero().flatten().tolist() == list(range(25, 35))
    out = ops.window_attention_native(**_to(case, gpu_device), window=10).cpu()
    assert out[:, :, lost].isnan().all()
    bound = ref.attention_bound(finite["query"], finite["key"], finite["value"], 0.0, 10, dtype, expected, True)
    _close(out[:, :, ~lost], expected[:, :, ~lost], bound[:, :, ~lost])
    for n in (25, 26, 35, 36):
        one = ops.window_attention_native(**_to({**case, "query": case["query"][:, :, :1]}, gpu_device), window=10,
                                          lengths=torch.tensor([n], device=gpu_device))
        assert bool(one.isnan().all()) == bool(lost[n - 1])


@pytest.mark.parametrize("scale", [2.0 ** -126, -(2.0 ** -126), 2.0 ** -103, 2.0 ** 103, 2.0 ** 120, 3e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_window_scales_next_to_what_float32_holds(gpu_device, dtype, scale):
    """Queries and keys that bring the scores back to ordinary ones, exactly: powers of two.  <q, k> is a float32 sum before
    the scale: from key 16 on it is j 2^124 >= 2^128 at the smallest scales, an infinite score."""
    case = {**_window_case(53, dtype, 1, 2, 1, 64, 40, 40), "scale": scale}
    each = 2.0 ** math.floor(-math.log2(abs(scale)) / 2)
    case["query"] = torch.full_like(case["query"], each)
    case["key"] = torch.zeros_like(case["key"])
    case["key"][0, 0, :, 3] = torch.arange(40.0) * each / 4
    raw = case["key"][0, 0, :, 3].double() * each
    bounded = {**case, "key": torch.where(raw.float().isinf()[:, None], 0.0, case["key"].double()).to(dtype)}
    scores = raw.float().double() * float(torch.tensor(scale))
    for window, sinks in ((0, 0), (9, 2)):
        expected = torch.zeros(1, 2, 40, 64, dtype=torch.float64)
        for i in range(40):
            seen = ref.visible_keys(i, 40, window, sinks)
            weights = torch.exp(scores[seen] - scores[seen].max())
            expected[0, :, i] = weights @ case["value"][0, 0, seen].double() / weights.sum()
        lost = expected.isnan()
        assert bool(lost.any()) == (scale == 2.0 ** -126)
        out = ops.window_attention_native(**_to(case, gpu_device), window=window, sinks=sinks).cpu()
        assert torch.equal(out.isnan(), lost)
        bound = ref.attention_bound(bounded["query"], bounded["key"], bounded["value"], scale, 40, dtype, expected, True)
        _close(out.nan_to_num(), expected.nan_to_num(), bound.nan_to_num())


@pytest.mark.parametrize("dtype", TYPES)
def test_window_padded_batches_and_chunks(gpu_device, dtype):
    case = _window_case(9, dtype, 5, 6, 2, 64, 70, 70)
    out = _check_window(case, gpu_device, 16, 2, lengths=[70, 1, 0, 33, 64], starts=[0] * 5)
    assert not out[2].any() and not out[3, :, 33:].any()
    # Chunks of longer prompts; positions before the first and behind the last key see nothing.
    case = _window_case(10, dtype, 5, 6, 2, 64, 20, 100)
    _check_window(case, gpu_device, 16, 2, lengths=[100, 37, 20, 90, 500], starts=[80, 17, 0, 85, -5])
    _check_window(case, gpu_device, 16, 2, lengths=[100, 12, 0, 90, -3])
    _check_window(case, gpu_device, 0, 0, lengths=[100] * 5, starts=[-(2 ** 62), 2 ** 62, 99, -19, -20])
    case = _window_case(12, dtype, 5, 6, 2, 64, 1, 100)
    _check_window(case, gpu_device, 16, 2, lengths=[100, 37, 0, 90, 500], starts=[50, 36, 0, 90, -1])


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 128)])
def test_window_longer_prompts(gpu_device, dtype, dim):
    """Against the formula in float64 as one product on the CPU, many tiles deep."""
    case = _window_case(21, dtype, 1, 6, 2, dim, 1500, 1500)
    for window, sinks in ((256, 4), (0, 0)):
        p, j = torch.arange(1500)[:, None], torch.arange(1500)
        seen = (j <= p) & ((j > p - window) | (j < sinks) if window else j >= 0)
        keys, values = (case[k].double().repeat_interleave(3, dim=1) for k in ("key", "value"))
        scores = (case["query"].double() @ keys.transpose(2, 3) * case["scale"]).masked_fill(~seen, -math.inf)
        expected = torch.softmax(scores, -1) @ values
        actual = ops.window_attention_native(**_to(case, gpu_device), window=window, sinks=sinks)
        _close(actual, expected, ref.attention_bound(case["query"], case["key"], case["value"], case["scale"], 1500, dtype,
                                                     expected, True))


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 64), (torch.float16, 128)])
def test_window_strides(gpu_device, dtype, dim):
    case = _to(_window_case(25, dtype, 2, 6, 2, dim, 70, 70), gpu_device)
    expected = ops.window_attention_native(**case, window=30, sinks=2)
    rows = {k: case[k].transpose(1, 2).contiguous().transpose(1, 2) for k in ("query", "key", "value")}
    assert torch.equal(ops.window_attention_native(**rows, scale=case["scale"], window=30, sinks=2), expected)
    odd = dict(rows)
    for name in ("key", "value"):
        store = torch.randn(2, 2, 70, dim + 3, device=gpu_device).to(dtype)
        store[..., 1:dim + 1] = case[name]
        odd[name] = store[..., 1:dim + 1]
    odd["query"] = case["query"].transpose(1, 3).contiguous().transpose(1, 3)
    assert torch.equal(ops.window_attention_native(**odd, scale=case["scale"], window=30, sinks=2), expected)
    # One key row for all positions (a stride of zero) is a broadcast like any other.
    one = {k: case[k][:, :, :1].expand(2, 2, 70, dim) for k in ("key", "value")}
    out = ops.window_attention_native(case["query"], **one, scale=case["scale"], window=30, sinks=2)
    torch.testing.assert_close(out, one["value"].repeat_interleave(3, 1).contiguous(), rtol=2 * torch.finfo(dtype).eps, atol=1e-6)


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 64)])
def test_window_nan_reaches_only_the_rows_that_see_it(gpu_device, dtype, dim):
    case = _window_case(27, dtype, 1, 4, 2, dim, 120, 120)
    window, sinks = 16, 2
    clean = ops.window_attention_native(**_to(case, gpu_device), window=window, sinks=sinks).cpu()
    for name in ("key", "value"):
        for bad, at in ((math.nan, 50), (math.inf, 51), (-math.inf, 1), (math.nan, 119)):
            dirty = {**case, name: case[name].clone()}
            dirty[name][0, 0, at, 3] = bad
            out = ops.window_attention_native(**_to(dirty, gpu_device), window=window, sinks=sinks).cpu()
            expected = ref.window_attention(**dirty, window=window, sinks=sinks)
            assert torch.equal(out[0, 2:], clean[0, 2:])
            for i in range(120):
                if at not in ref.visible_keys(i, 120, window, sinks):
                    _close(out[0, :2, i], expected[0, :2, i], ref.attention_bound(
                        case["query"], case["key"], case["value"], case["scale"], window + sinks, dtype, expected[0, :2, i], True))
                else:
                    assert torch.equal(out[0, :2, i].isnan(), expected[0, :2, i].isnan()), (name, bad, at, i)


def test_window_rows_that_are_all_nan(gpu_device):
    case = _to(_window_case(29, torch.bfloat16, 1, 4, 2, 64, 700, 700), gpu_device)
    for name in ("key", "value"):
        dirty = {**case, name: torch.full_like(case[name], math.nan)}
        assert bool(ops.window_attention_native(**dirty, window=300, sinks=2).isnan().all())
    half = {**case, "value": case["value"].clone()}
    half["value"][..., ::2] = math.inf  # every dim of every row sees one; the others stay finite
    out = ops.window_attention_native(**half, window=300, sinks=2)
    assert bool(out[..., 1::2].isfinite().all()) and not bool(out[..., ::2].isfinite().any())


def test_window_other_stream_and_graph(gpu_device):
    case = _to(_window_case(33, torch.bfloat16, 2, 8, 2, 64, 90, 90), gpu_device)
    lengths, starts = torch.tensor([90, 40], device=gpu_device), torch.zeros(2, dtype=torch.int64, device=gpu_device)
    expected = ops.window_attention_native(**case, window=20, lengths=lengths, starts=starts)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = ops.window_attention_native(**case, window=20, lengths=lengths, starts=starts)
    torch.cuda.synchronize()
    assert torch.equal(other, expected)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.window_attention_native(**case, window=20, lengths=lengths, starts=starts)
    for n in (40, 77, 1):
        lengths[1] = n
        case["query"].mul_(0.5)
        graph.replay()
        assert torch.equal(captured, ops.window_attention_native(**case, window=20, lengths=lengths, starts=starts))


# --------------------------------------------------------------------------- pages

class _Device:
    """The pages of ``ref.Pages`` on the GPU, next to it."""

    def __init__(self, model, device):
        self.model, self.device = model, device
        self.key, self.value = model.key.to(device), model.value.to(device)
        self.table = torch.tensor(model.table, dtype=torch.int32, device=device)
        self.lengths = torch.tensor(model.lengths, device=device)
        self.refcounts = torch.tensor(model.refcounts, dtype=torch.int32, device=device)

    @property
    def books(self):
        return self.table, self.lengths, self.refcounts

    def ids(self, values):
        return torch.tensor(values, dtype=torch.int64, device=self.device)

    def same(self):
        assert self.table.tolist() == self.model.table
        assert self.lengths.tolist() == self.model.lengths
        assert self.refcounts.tolist() == self.model.refcounts
        assert torch.equal(self.key.cpu(), self.model.key) and torch.equal(self.value.cpu(), self.model.value)

    def reserve(self, slots, counts):
        positions, status = ops.paged_cache_reserve_native(*self.books, self.model.page_size, self.ids(slots), self.ids(counts))
        assert (positions.tolist(), status.tolist()) == self.model.reserve(slots, counts)
        return positions

    def write(self, layer, key, value, slots, positions, counts):
        ops.paged_cache_write_native(key.to(self.device), value.to(self.device), self.key[layer], self.value[layer],
                                     self.table, self.ids(slots), positions, self.ids(counts))
        self.model.write(layer, key, value, slots, positions.tolist(), counts)

    def copy(self, source, target):
        status = ops.paged_cache_copy_native(self.key, self.value, self.ids(source), self.ids(target))
        assert status.tolist() == self.model.copy(source, target)

    def free(self, slots):
        assert ops.paged_cache_free_native(*self.books, self.ids(slots)).tolist() == self.model.free(slots)

    def fork(self, parents, children):
        status = ops.paged_cache_fork_native(self.key, self.value, *self.books, self.ids(parents), self.ids(children))
        expected = self.model.fork(parents, children)
        assert status.tolist() == expected
        return expected

    def compact(self):
        page_map, used = ops.paged_cache_compact_native(self.key, self.value, self.table, self.refcounts)
        assert (page_map.tolist(), int(used)) == self.model.compact()


@pytest.mark.parametrize("dtype,dim,page_size,layers", [(torch.float32, 64, 16, 2), (torch.bfloat16, 40, 5, 3),
                                                        (torch.float16, 7, 3, 1), (torch.float32, 3, 1, 2)])
def test_pages_in_random_order(gpu_device, dtype, dim, page_size, layers):
    """Every operator against the lists, requests out of range, repeated and beyond the pool among them."""
    rng = random.Random(dim)
    slots, columns = 9, 6
    model = ref.Pages(layers, 24, 2, page_size, dim, slots, columns, dtype, seed=dim)
    pages = _Device(model, gpu_device)
    g = torch.Generator().manual_seed(1)
    seen = set()
    for _ in range(120):
        action = rng.choice(("grow", "grow", "grow", "fork", "free", "compact", "copy"))
        count = rng.randint(1, 5)
        some = [rng.randint(-1, slots) for _ in range(count)]
        if action == "grow":
            counts = [rng.choice((0, 1, 1, page_size, 2 * page_size + 1, -1)) for _ in some]
            positions = pages.reserve(some, counts)
            key, value = (torch.randn(count, 2, 2 * page_size + 1, dim, generator=g).to(dtype) for _ in range(2))
            for layer in range(layers):
                pages.write(layer, key, value, some, positions, counts)
        elif action == "fork":
            seen |= set(pages.fork(some, [rng.randint(-1, slots) for _ in some]))
        elif action == "free":
            pages.free(some)
        elif action == "compact":
            pages.compact()
        else:
            pages.copy([rng.randint(-1, 24) for _ in some], [rng.randint(0, 24) for _ in some])
        pages.same()
    assert {ref.DONE, ref.OUT_OF_RANGE, ref.OCCUPIED} <= seen


def test_pages_of_large_pools_and_many_requests(gpu_device):
    """Pools and lists longer than one round of the bookkeeping workgroup, with every lowest page taken in order."""
    model = ref.Pages(1, 9001, 1, 2, 1, 2500, 4)
    rng = random.Random(3)
    for p in range(9001):
        model.refcounts[p] = rng.choice((0, 0, 1))
    pages = _Device(model, gpu_device)
    order = list(range(2500))
    rng.shuffle(order)
    pages.reserve(order, [rng.randint(0, 8) for _ in order])
    pages.same()
    parents = [s for s in order if model.lengths[s]][:900]
    empty = [s for s in order if not model.lengths[s]]
    pages.free(order[-300:])
    pages.fork(parents[: len(empty)], empty[: len(parents)])
    pages.same()
    pages.compact()
    pages.same()
    pages.free(order)
    pages.same()


def test_pages_run_out_in_order(gpu_device):
    pages = _Device(ref.Pages(2, 5, 1, 4, 8, 6, 4), gpu_device)
    pages.reserve([0, 1, 2, 3, 4], [8, 3, 9, 0, 1])  # 2 + 1 pages fit, the third asks for 3, and the last for 1 more
    assert pages.lengths.tolist() == [8, 3, 0, 0, 0, 0]
    pages.reserve([1, 0], [1, 9])  # a page in hand; a row that is too short
    pages.same()
    pages.reserve([2, 3], [4, 4])
    assert pages.fork([1, 0, 1], [4, 5, 4]) == [ref.DONE, ref.DONE, ref.REPEATED]  # full pages only: none is needed
    pages.free([4])
    pages.reserve([1], [1])
    pages.same()
    # A chain in one call reads the books as they were: slot 4 is empty as a parent.
    assert pages.fork([0, 4], [4, 4]) == [ref.DONE, ref.REPEATED]
    pages.same()


def test_page_copies_that_clash_are_refused(gpu_device):
    pages = _Device(ref.Pages(3, 8, 2, 4, 16, 1, 1), gpu_device)
    pages.copy([0, 1, 2, 2, 5, 7, -1, 0], [1, 3, 4, 4, 5, 8, 6, 6])
    pages.same()
    assert ops.paged_cache_copy_native(pages.key, pages.value, pages.ids([]), pages.ids([])).shape == (0,)


def test_pages_with_other_strides(gpu_device):
    """Pools as views of [layers, P, page, heads, D] and of one tensor for keys and values; rows that are not aligned."""
    model = ref.Pages(2, 8, 3, 4, 6, 4, 3, torch.float32, seed=2)
    pages = _Device(model, gpu_device)
    both = torch.zeros(2, 2, 8, 4, 3, 7, device=gpu_device)
    untouched = both[..., 6].clone().fill_(5.0)
    both[..., 6] = untouched
    views = both[0, ..., :6].transpose(2, 3), both[1, ..., :6].transpose(2, 3)
    for view, source in zip(views, (pages.key, pages.value)):
        view.copy_(source)
    pages.key, pages.value = views
    table = torch.full((4, 5), 77, dtype=torch.int32, device=gpu_device)
    table[:, 1:4] = -1
    pages.table = table[:, 1:4]
    positions = pages.reserve([2, 0], [10, 5])
    for layer in range(2):
        key = torch.randn(2, 10, 3, 6).transpose(1, 2)
        pages.write(layer, key, -key, [2, 0], positions, [10, 5])
    pages.fork([2, 0], [1, 3])
    pages.free([2])
    pages.compact()
    pages.copy([0], [7])
    pages.same()
    assert torch.equal(both[..., 6], untouched) and bool((table[:, [0, 4]] == 77).all())


def test_pools_of_one_storage(gpu_device):
    """Interleaved keys and values work as separate ones; views that meet are refused before any launch."""
    shape = (3, 9, 2, 4, 8)
    ids = torch.tensor([0, 4, 7], device=gpu_device)
    source = torch.randn(2, *shape, generator=torch.Generator().manual_seed(3)).to(gpu_device)
    expected = source.clone()
    expected[:, :, ids + 1] = source[:, :, ids]
    for layout in ((3, 9, 2, 2, 4, 8), (3, 9, 2, 4, 2, 8)):
        at = layout.index(2, 2) if layout[3] == 2 else 4
        store = torch.zeros(layout, device=gpu_device)
        key, value = store.unbind(at)
        key.copy_(source[0]), value.copy_(source[1])
        status = ops.paged_cache_copy_native(key, value, ids, ids + 1)
        assert status.tolist() == [ops.PAGE_DONE] * 3
        assert torch.equal(key, expected[0]) and torch.equal(value, expected[1])
    store = torch.randn(3 * 9 * 64 + 64, device=gpu_device)
    key, value = store[:-64].view(shape), store[64:].view(shape)
    books = {"page_table": torch.full((3, 4), -1, dtype=torch.int32, device=gpu_device),
             "lengths": torch.zeros(3, dtype=torch.int64, device=gpu_device),
             "refcounts": torch.zeros(9, dtype=torch.int32, device=gpu_device)}
    rows = torch.zeros(1, 2, 1, 8, device=gpu_device)
    kept = store.clone()
    for call in (lambda: ops.paged_cache_copy_native(key, value, ids, ids + 1),
                 lambda: ops.paged_cache_fork_native(key, value, *books.values(), ids[:1], ids[:1] + 1),
                 lambda: ops.paged_cache_compact_native(key, value, books["page_table"], books["refcounts"]),
                 lambda: ops.paged_cache_write_native(rows, rows.clone(), key[0], value[0], books["page_table"], ids[:1], ids[:1])):
        with pytest.raises(RuntimeError, match="key and value pages must not overlap"):
            call()
    assert torch.equal(store, kept)


def test_write_skips_what_has_no_page(gpu_device):
    pages = _Device(ref.Pages(1, 4, 1, 4, 8, 3, 2), gpu_device)
    pages.table[0, 0] = pages.model.table[0][0] = 2
    pages.table[1, 0] = pages.model.table[1][0] = 9  # outside the pool
    key = torch.randn(4, 1, 9, 8)
    pages.write(0, key, -key, [0, 1, 3, 2], pages.ids([1, 0, 0, -1]), [9, 9, 9, 9])
    pages.same()
    pages.write(0, key[:1], key[:1], [0], pages.ids([2 ** 62]), [9])
    pages.same()


# --------------------------------------------------------------------------- logits

def _logits_case(seed, dtype, rows, vocab, width, bias_rows=1, allowed_rows=None):
    g = torch.Generator().manual_seed(seed)
    history = torch.randint(0, vocab, (rows, width), generator=g)
    history[:, ::3] %= min(vocab, 5)
    return {"logits": (3 * torch.randn(rows, vocab, generator=g)).to(dtype), "history": history,
            "history_lengths": torch.randint(0, width + 1, (rows,), generator=g),
            "repetition": 1 + torch.rand(rows, generator=g), "frequency": torch.rand(rows, generator=g),
            "presence": torch.rand(rows, generator=g), "bias": torch.randn(bias_rows, vocab, generator=g),
            "allowed": torch.randint(-2 ** 31, 2 ** 31, (allowed_rows or rows, -(-vocab // 32)), generator=g).to(torch.int32)}


def _check_logits(case, device):
    expected = ref.processed_logits(**case)
    processed, tokens = ops.logits_process_native(**_to(case, device))
    assert processed.dtype == case["logits"].dtype and tokens.dtype == torch.int64
    cpu = processed.cpu()
    assert torch.equal(cpu.isneginf(), expected.isneginf()) and torch.equal(cpu.isnan(), expected.isnan())
    fine = expected.isfinite()
    # Five float32 roundings of intermediate values that are at most the sum of the magnitudes, one to the type.
    size = case["logits"].double().abs() * 2
    for name in ("frequency", "presence"):
        if case.get(name) is not None:
            size = size + case[name].double()[:, None] * (case["history"].shape[1] if name == "frequency" else 1)
    if case.get("bias") is not None:
        size = size + case["bias"].double().abs()
    bound = 5 * 2.0 ** -24 * size + torch.finfo(case["logits"].dtype).eps / 2 * expected.abs().nan_to_num(posinf=0)
    error = (cpu.double() - expected).abs()
    assert bool((error[fine] <= bound.expand_as(error)[fine] + torch.finfo(case["logits"].dtype).tiny).all())
    assert tokens.tolist() == ref.greedy(cpu)
    return cpu, tokens


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 1000, 8191, 8192, 8193, 20001, 49152])
def test_logits_sizes(gpu_device, dtype, vocab):
    _check_logits(_logits_case(vocab, dtype, 3, vocab, 50), gpu_device)
    _check_logits(_logits_case(vocab + 1, dtype, 1, vocab, 1, allowed_rows=1), gpu_device)


def test_logits_options(gpu_device):
    case = _logits_case(1, torch.float32, 4, 5000, 600, bias_rows=4, allowed_rows=1)
    _check_logits(case, gpu_device)
    names = ("history_lengths", "repetition", "frequency", "presence", "bias", "allowed")
    for left_out in names:
        _check_logits({k: v for k, v in case.items() if k != left_out}, gpu_device)
    for alone in names:
        _check_logits({k: v for k, v in case.items() if k in ("logits", "history", alone)}, gpu_device)
    plain, tokens = _check_logits({"logits": case["logits"]}, gpu_device)
    assert torch.equal(plain, case["logits"]) and tokens.tolist() == case["logits"].argmax(1).tolist()
    _check_logits({**case, "history": torch.zeros(4, 0, dtype=torch.int64), "history_lengths": None}, gpu_device)


def test_logits_edges(gpu_device):
    """Padding ids, lengths outside the width, ties, rows that allow nothing, NaN and infinity, also where masked."""
    case = _logits_case(2, torch.float32, 6, 9000, 40)
    case["history"][0, 5:] = -1
    case["history"][1, :] = 2 ** 40
    case["history_lengths"] = torch.tensor([40, 40, 0, 100, -1, 7])
    case["allowed"][2] = 0
    case["logits"][3] = 1.5
    case["logits"][4, 100] = math.nan
    case["logits"][4, 8999] = math.nan
    case["logits"][5, :50] = torch.tensor([math.nan, math.inf, -math.inf, math.nan, 3.0] * 10)
    case["allowed"][4, 3] |= 1 << 4
    case["allowed"][4, 8999 // 32] |= 1 << (8999 % 32)
    _, tokens = _check_logits(case, gpu_device)
    assert int(tokens[2]) == 0 and int(tokens[4]) == 100
    case = {"logits": torch.zeros(2, 20000)}
    case["logits"][1, [15000, 300, 8192]] = 1.0
    assert _check_logits(case, gpu_device)[1].tolist() == [0, 300]
    low = torch.full((1, 100), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16)
    out, tokens = ops.logits_process_native(low.to(gpu_device), bias=torch.full((1, 100), -1e38, device=gpu_device))
    assert int(tokens[0]) == 0 and bool(out.cpu().isneginf().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 20000), (300, 8200), (300, 8203)])
def test_logits_ties_go_to_the_lowest_index(gpu_device, dtype, rows, vocab):
    """Zeros of both signs are equal, what a rounding makes equal is equal, and the first NaN is above all."""
    low = torch.full((rows, vocab), -3.0, dtype=dtype)
    for places in ([0, 1], [7, 8], [5, 4100], [2047, 2048], [4093, 8199], [vocab - 2, vocab - 1]):
        for first, second in ((0.0, -0.0), (-0.0, 0.0), (math.inf, math.inf), (math.nan, math.nan), (math.nan, math.inf)):
            logits = low.clone()
            logits[:, places[0]], logits[:, places[1]] = first, second
            processed, tokens = ops.logits_process_native(logits.to(gpu_device))
            assert tokens.tolist() == [places[0]] * rows, (places, first, second)
            assert torch.equal(processed.cpu().nan_to_num(nan=9.0), logits.nan_to_num(nan=9.0))
        # The second is larger by less than half a step of the type before the rounding.
        logits = low.clone()
        logits[:, places] = 1.0
        bias = torch.zeros(1, vocab)
        bias[0, places[1]] = torch.finfo(dtype).eps / 4
        _, tokens = ops.logits_process_native(logits.to(gpu_device), bias=bias.to(gpu_device))
        assert tokens.tolist() == [places[0]] * rows


@pytest.mark.parametrize("rows,vocab", [(1, 2 ** 24), (2, 2 ** 24 - 5), (70001, 5)])
def test_logits_of_the_largest_shapes(gpu_device, rows, vocab):
    g = torch.Generator().manual_seed(rows)
    logits = torch.randn(rows, vocab, generator=g).half()
    at = torch.randint(0, vocab, (rows,), generator=g)
    logits[torch.arange(rows), at] = 100.0
    history = torch.stack([at, (at + 1) % vocab], 1)
    processed, tokens = ops.logits_process_native(logits.to(gpu_device), history.to(gpu_device),
                                                  presence=torch.full((rows,), 0.5, device=gpu_device))
    assert torch.equal(tokens.cpu(), at)
    expected = logits.float()
    for column in range(2):
        expected[torch.arange(rows), history[:, column]] -= 0.5
    assert torch.equal(processed.cpu(), expected.half())


def test_logits_strides(gpu_device):
    case = _logits_case(3, torch.float16, 4, 4096, 64, bias_rows=4)
    device = _to(case, gpu_device)
    expected, tokens = ops.logits_process_native(**device)
    for name, extra in (("logits", 8), ("logits", 3), ("history", 5), ("bias", 3), ("bias", 4), ("allowed", 1)):
        wide = torch.zeros(4, device[name].shape[1] + extra, dtype=device[name].dtype, device=gpu_device)
        wide[:, : device[name].shape[1]] = device[name]
        moved = {**device, name: wide[:, : device[name].shape[1]]}
        out, again = ops.logits_process_native(**moved)
        assert torch.equal(out, expected) and torch.equal(again, tokens)
        shifted = torch.zeros(4, device[name].shape[1] + 8, dtype=device[name].dtype, device=gpu_device)
        shifted[:, 1:1 + device[name].shape[1]] = device[name]
        out, again = ops.logits_process_native(**{**device, name: shifted[:, 1:1 + device[name].shape[1]]})
        assert torch.equal(out, expected) and torch.equal(again, tokens)


def test_opcheck(gpu_device):
    case = _to(_paged_case(43, torch.float32, 6, 2, 64, 16, [50, 20]), gpu_device)
    for op, args in ((torch.ops.flux.paged_decode_attention.default, tuple(case.values())),
                     (torch.ops.flux.window_attention.default,
                      tuple(_to(_window_case(1, torch.float32, 2, 4, 2, 64, 5, 9), gpu_device).values()) + (4,)),
                     (torch.ops.flux.logits_process.default, (torch.randn(2, 100, device=gpu_device),))):
        result = torch.library.opcheck(op, args)
        assert all(status == "SUCCESS" for status in result.values()), result
    pages = _Device(ref.Pages(2, 9, 2, 4, 8, 3, 4), gpu_device)
    pools, ids = (pages.key, pages.value), pages.ids([0, 2])
    rows = torch.randn(2, 2, 3, 8, device=gpu_device)
    for op, args in ((torch.ops.flux.paged_cache_reserve, (*pages.books, 4, ids, pages.ids([3, 5]))),
                     (torch.ops.flux.paged_cache_write, (rows, -rows, pages.key[0], pages.value[0], pages.table, ids, ids)),
                     (torch.ops.flux.paged_cache_copy, (*pools, ids, ids + 1)),
                     (torch.ops.flux.paged_cache_fork, (*pools, *pages.books, ids[:1], ids[:1] + 1)),
                     (torch.ops.flux.paged_cache_free, (*pages.books, ids)),
                     (torch.ops.flux.paged_cache_compact, (*pools, pages.table, pages.refcounts))):
        result = torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))
        assert all(status == "SUCCESS" for status in result.values()), result


# --------------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", TYPES)
def test_a_served_loop(gpu_device, dtype):
    """Prompts through the window operator and into pages, branches, decoded tokens, upkeep of the pool between them: each
    step's attention against the whole history in float64, and the tokens against the plain logits."""
    g = torch.Generator().manual_seed(51)
    layers, heads, kv_heads, dim, page_size, window, sinks, vocab = 2, 6, 2, 64, 16, 24, 2, 500
    pages = _Device(ref.Pages(layers, 40, kv_heads, page_size, dim, 6, 8, dtype), gpu_device)
    prompts = [37, 16, 5]
    history = {}  # slot -> per layer (keys, values), tokens
    slots = [4, 0, 2]
    width = max(prompts)
    positions = pages.reserve(slots, prompts)
    layer_rows = [[_randn(g, (3, kv_heads, width, dim), dtype) for _ in range(2)] for _ in range(layers)]
    for layer, (key, value) in enumerate(layer_rows):
        query = _randn(g, (3, heads, width, dim), dtype)
        _check_window({"query": query, "key": key, "value": value, "scale": 0.125}, gpu_device, window, sinks,
                      lengths=prompts, starts=[0, 0, 0])
        pages.write(layer, key, value, slots, positions, prompts)
    for i, slot in enumerate(slots):
        history[slot] = ([(k[i, :, : prompts[i]], v[i, :, : prompts[i]]) for k, v in layer_rows], [i, i, 7])
    assert pages.fork([4, 0], [1, 5]) == [ref.DONE, ref.DONE]
    for parent, child in ((4, 1), (0, 5)):
        history[child] = (list(history[parent][0]), list(history[parent][1]))
    for step in range(20):
        active = sorted(history)
        ids = pages.ids(active)
        positions = pages.reserve(active, [1] * len(active))
        assert min(positions.tolist()) >= 0
        for layer in range(layers):
            key, value = (_randn(g, (len(active), kv_heads, 1, dim), dtype) for _ in range(2))
            query = _randn(g, (len(active), heads, 1, dim), dtype)
            pages.write(layer, key, value, active, positions, [1] * len(active))
            out = ops.paged_decode_attention_native(query.to(gpu_device), pages.key[layer], pages.value[layer], pages.table,
                                                    pages.lengths, 0.125, window, sinks, ids)
            for i, slot in enumerate(active):
                keys, values = history[slot][0][layer]
                keys, values = torch.cat((keys, key[i]), 1), torch.cat((values, value[i]), 1)
                history[slot][0][layer] = (keys, values)
                expected = ref.window_attention(query[i][None], keys[None], values[None], 0.125, window, sinks)
                _close(out[i][None], expected, ref.attention_bound(query[i], keys, values, 0.125, window + sinks, dtype, expected))
        logits = torch.randn(len(active), vocab, generator=g).to(dtype)
        past = torch.full((len(active), 40), -1)
        for i, slot in enumerate(active):
            past[i, : len(history[slot][1])] = torch.tensor(history[slot][1])
        rate = torch.full((len(active),), 1.3)
        _, tokens = _check_logits({"logits": logits, "history": past, "repetition": rate, "presence": rate}, gpu_device)
        for slot, token in zip(active, tokens.tolist()):
            history[slot][1].append(token)
        if step == 6:
            pages.free([0])
            del history[0]
            pages.compact()
        if step == 11:
            assert pages.fork([1], [3]) == [ref.DONE]
            history[3] = (list(history[1][0]), list(history[1][1]))
        pages.same()


def test_a_decode_step_in_a_graph(gpu_device):
    """Reserve, write, attend and pick the token as one captured graph, replayed with the program's own work between."""
    g = torch.Generator().manual_seed(61)
    model = ref.Pages(1, 30, 2, 4, 64, 3, 9)
    pages = _Device(model, gpu_device)
    positions = pages.reserve([0, 1, 2], [5, 1, 8])
    rows = torch.randn(3, 2, 8, 64, generator=g)
    pages.write(0, rows, -rows, [0, 1, 2], positions, [5, 1, 8])
    slots = pages.ids([2, 0, 1])
    key, value, query = (torch.zeros(3, h, 1, 64, device=gpu_device) for h in (2, 2, 4))
    history = torch.full((3, 30), -1, dtype=torch.int64, device=gpu_device)
    logits = torch.zeros(3, 9000, device=gpu_device)
    rate = torch.full((3,), 1.2, device=gpu_device)

    def step():
        at, status = ops.paged_cache_reserve_native(*pages.books, 4, slots)
        ops.paged_cache_write_native(key, value, pages.key[0], pages.value[0], pages.table, slots, at)
        out = ops.paged_decode_attention_native(query, pages.key[0], pages.value[0], pages.table, pages.lengths, 0.125, 6, 1, slots)
        processed, tokens = ops.logits_process_native(logits, history, None, rate)
        return at, status, out, processed, tokens

    books = [t.clone() for t in (*pages.books, pages.key, pages.value)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    for t, before in zip((*pages.books, pages.key, pages.value), books):
        t.copy_(before)
    with torch.cuda.graph(graph):
        captured = step()
    for t, before in zip((*pages.books, pages.key, pages.value), books):
        t.copy_(before)
    for i in range(9):
        for t in (key, value, query, logits):
            t.copy_(torch.randn(t.shape, generator=g))
        history[:, i] = i
        before = [t.clone() for t in (*pages.books, pages.key, pages.value)]
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured] + [t.clone() for t in (*pages.books, pages.key, pages.value)]
        for t, old in zip((*pages.books, pages.key, pages.value), before):
            t.copy_(old)
        eager = [*step(), *pages.books, pages.key, pages.value]
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), i


def test_two_graphs_replayed_in_turn(gpu_device):
    """Captured calls keep workspaces of their own: cut sequences, single windowed tokens, logits and pages in two graphs."""
    cases = [_to(_paged_case(67 + i, torch.float32, 6, 2, 64, 16, [3000 - 900 * i, 700, 40]), gpu_device) for i in range(2)]
    rows = [_to(_window_case(71 + i, torch.bfloat16, 2, 4, 2, 64, 1, 2500), gpu_device) for i in range(2)]
    logits = [torch.randn(2, 20000, generator=torch.Generator().manual_seed(73 + i)).to(gpu_device) for i in range(2)]
    books = [(torch.full((3, 4), -1, dtype=torch.int32, device=gpu_device), torch.zeros(3, dtype=torch.int64, device=gpu_device),
              torch.zeros(9 + i, dtype=torch.int32, device=gpu_device)) for i in range(2)]
    slots = torch.tensor([2, 0], device=gpu_device)

    def step(i):
        at, status = ops.paged_cache_reserve_native(*books[i], 4, slots)
        return (ops.paged_decode_attention_native(**cases[i], window=0), ops.window_attention_native(**rows[i], window=2000, sinks=3),
                *ops.logits_process_native(logits[i]), at, status)

    graphs, outputs = [], []
    for i in range(2):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(i)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs.append(step(i))
        graphs.append(graph)
    for turn in range(6):
        for case, row, logit in zip(cases, rows, logits):
            case["query"].normal_()
            row["query"].normal_()
            logit.normal_()
        for table, lengths, refcounts in books:
            table.fill_(-1)
            lengths.fill_(turn)
            refcounts.zero_()
        for i in ((0, 1), (1, 0))[turn % 2]:
            graphs[i].replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in (*outputs[i], *books[i])] for i in range(2)]
        for i in range(2):
            table, lengths, refcounts = books[i]
            table.fill_(-1)
            lengths.fill_(turn)
            refcounts.zero_()
            eager = [*step(i), *books[i]]
            assert all(torch.equal(a, b) for a, b in zip(got[i], eager)), (turn, i)


def test_offsets_beyond_32_bits(gpu_device):
    """A pool of more than 2^32 elements gives what a small one gives, and so do rows far apart."""
    dim, page_size, far = 128, 64, 2 ** 32 // (128 * 64)
    small = [torch.zeros(12, 1, page_size, dim, dtype=torch.bfloat16, device=gpu_device) for _ in range(2)]
    large = [torch.empty(far + 12, 1, page_size, dim, dtype=torch.bfloat16, device=gpu_device) for _ in range(2)]
    for pool in large:
        pool[far:] = 0
    key, value = (torch.randn(2, 1, 150, dim, device=gpu_device).bfloat16() for _ in range(2))
    query = torch.randn(3, 4, 1, dim, device=gpu_device).bfloat16()
    slots, counts = torch.tensor([0, 1], device=gpu_device), torch.tensor([150, 70], device=gpu_device)
    source, target = torch.tensor([0, 3], device=gpu_device), torch.tensor([9, 10], device=gpu_device)
    results = []
    for (key_pages, value_pages), start in ((small, 0), (large, far)):
        table = torch.full((3, 4), -1, dtype=torch.int32, device=gpu_device)
        lengths = torch.zeros(3, dtype=torch.int64, device=gpu_device)
        refcounts = torch.zeros(start + 12, dtype=torch.int32, device=gpu_device)
        refcounts[:start] = 1
        positions, status = ops.paged_cache_reserve_native(table, lengths, refcounts, page_size, slots, counts)
        ops.paged_cache_write_native(key, value, key_pages, value_pages, table, slots, positions, counts)
        forked = ops.paged_cache_fork_native(key_pages, value_pages, table, lengths, refcounts, slots[:1], slots[:1] + 2)
        copied = ops.paged_cache_copy_native(key_pages, value_pages, source + start, target + start)
        out = ops.paged_decode_attention_native(query, key_pages, value_pages, table, lengths, dim ** -0.5)
        results.append([status, positions, forked, copied, out, lengths, torch.where(table >= 0, table - start, table),
                        refcounts[start:], key_pages[start:], value_pages[start:]])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert bool(results[0][4].any()) and results[0][0].tolist() == [0, 0]
    # A page from behind 2^32 elements to the front.
    held = large[0][far + 1].clone()
    free = torch.ones(far + 12, dtype=torch.int32, device=gpu_device)
    free[far + 2 :] = 0
    free[5] = free[6] = 0
    table = torch.tensor([[far, far + 1]], dtype=torch.int32, device=gpu_device)
    page_map, used = ops.paged_cache_compact_native(*large, table, free)
    assert int(used) == far and table.tolist() == [[5, 6]] and page_map[far:].tolist() == [5, 6] + [-1] * 10
    assert torch.equal(large[0][6], held)
    # Rows 2^23 elements apart, and sequences 2^31: keys and values side by side.
    flat, apart, sequence = large[0].view(-1), 2 ** 23, 2 ** 31 + 64
    case = _to(_window_case(79, torch.bfloat16, 2, 4, 1, dim, 200, 250), gpu_device)
    spread = {"key": flat.as_strided((2, 1, 250, dim), (sequence, dim, apart, 1)),
              "value": flat.as_strided((2, 1, 250, dim), (sequence, dim, apart, 1), dim)}
    for name, view in spread.items():
        view.copy_(case[name])
    for queries in (1, 200):
        q = case["query"][:, :, :queries]
        expected = ops.window_attention_native(**{**case, "query": q}, window=90, sinks=5)
        assert torch.equal(ops.window_attention_native(q, **spread, scale=case["scale"], window=90, sinks=5), expected)
