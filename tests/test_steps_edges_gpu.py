"""Mixed steps where parts of a tile, or numbers next to a limit, could go another way than the whole (``oracle/steps.py``)."""

from __future__ import annotations

import math

import pytest
import torch

from flux_amd import ops
from oracle import steps
from tests.test_steps_gpu import TYPES, _bound, _check_chunk, _check_sample, _chunk_case, _close, _to

pytestmark = pytest.mark.gpu

# Heads, KV heads, head dimension, tokens of the one request, keys before them: tiles in two parts and more (at most 4, 8, and
# beyond), float32 on its own instruction and, from 2048 rows on, in limbs.
CUT = [(4, 2, 64, 1, 700), (4, 2, 64, 3, 1100), (4, 2, 128, 1, 600), (4, 2, 128, 20, 1500), (4, 1, 80, 1, 4400), (2, 1, 256, 5, 900),
       (32, 1, 64, 70, 400), (32, 1, 40, 70, 3000), (1, 1, 64, 1, 20000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,tokens,before", CUT)
def test_nan_that_fills_a_part_reaches_the_row(gpu_device, dtype, heads, kv_heads, dim, tokens, before):
    """Three quarters of the keys are NaN, so that whole parts have no other score: every row that sees one is NaN."""
    case = _chunk_case(dim + before, dtype, heads, kv_heads, dim, 16, [(tokens, before)])
    pages = case["page_table"][0, : before * 3 // 4 // 16].long()
    case["key_pages"][pages] = math.nan
    expected = steps.chunk_attention(**case)
    assert bool(expected.isnan().all())
    assert bool(ops.paged_chunk_attention_native(**_to(case, gpu_device)).isnan().all())
    # The token's own key alone.
    case = _chunk_case(dim + before, dtype, heads, kv_heads, dim, 16, [(1, before // 64 * 64)])
    case["key_pages"][case["page_table"][0, before // 64 * 4].long(), :, 0] = math.nan
    assert bool(ops.paged_chunk_attention_native(**_to(case, gpu_device)).isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,tokens,before", CUT)
@pytest.mark.parametrize("score", [-300.0, -math.inf])
def test_nan_and_infinite_values_behind_no_weight_reach_the_row(gpu_device, dtype, heads, kv_heads, dim, tokens, before, score):
    """0 times NaN or infinity is NaN, also where a whole part's weights are 0 next to another's: scores 300 below, and -inf."""
    case = _chunk_case(dim + before + 1, dtype, heads, kv_heads, dim, 16, [(tokens, before)], scale=0.125)
    case["query"][..., 0] = 1
    table = case["page_table"][0].long()
    pages = table[: before * 3 // 4 // 16]
    case["key_pages"][table, :, :, 0] = 0
    case["key_pages"][pages, :, :, 0] = 8 * score
    clean = {**case, "value_pages": case["value_pages"].clone(), "key_pages": case["key_pages"].nan_to_num(neginf=-2400)}
    for bad in (math.nan, math.inf):
        case["value_pages"][pages[3], :, 5, dim // 2] = bad
        actual = ops.paged_chunk_attention_native(**_to(case, gpu_device)).cpu()
        assert not bool(actual[..., dim // 2].isfinite().any())
    expected = steps.chunk_attention(**clean)
    kept = [d for d in range(dim) if d != dim // 2]
    close = {**clean, "key_pages": case["key_pages"].clamp(min=-64).nan_to_num()}  # the far ones' scores are no term
    _close(actual[..., kept], expected[..., kept], _bound(close, expected)[..., kept])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,tokens,before", CUT)
def test_rows_that_see_nothing_stay_zero_next_to_nan(gpu_device, dtype, heads, kv_heads, dim, tokens, before):
    """In cut tiles: a token before the first key, and a request whose pages are all gone (NaN stands for what is not its own)."""
    case = _chunk_case(dim + before + 2, dtype, heads, kv_heads, dim, 16, [(tokens, before)])
    case["key_pages"][case["page_table"][0, :2].long()] = math.nan
    case["value_pages"][case["page_table"][0, :2].long()] = math.nan
    positions = torch.tensor([-1])
    expected = steps.chunk_attention(**case, positions=positions)
    actual = ops.paged_chunk_attention_native(**_to(case, gpu_device), positions=positions.to(gpu_device)).cpu()
    assert not bool(actual[0].any()) and torch.equal(actual.isnan(), expected.isnan())
    gone = {**case, "key_pages": torch.full_like(case["key_pages"], math.nan), "value_pages": torch.full_like(case["key_pages"], math.nan),
            "page_table": torch.full_like(case["page_table"], -1)}
    assert not bool(ops.paged_chunk_attention_native(**_to(gone, gpu_device)).any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,tokens,before", CUT)
@pytest.mark.parametrize("size", [11.0, 2.0 ** 8, 2.0 ** 9, 2.0 ** 10, 2.0 ** 12])
def test_scores_that_are_exact_count_exactly(gpu_device, dtype, heads, kv_heads, dim, tokens, before, size):
    """Scores of 121, 2^16 to 2^24 and a few, exact in float32, that rise along the keys: the maximum moves, and what was summed
    before has to keep its weight."""
    case = _chunk_case(dim + before + 3, dtype, heads, kv_heads, dim, 16, [(tokens, before)], scale=1.0)
    case["query"].zero_()[..., 0] = size
    case["query"][..., 1] = 1
    key, n = case["key_pages"], tokens + before
    key.nan_to_num_().zero_()
    key[..., 0] = size
    rise = (torch.arange(n) * 64 // n).to(dtype)  # by one, 64 times
    at = torch.arange(n)
    key[case["page_table"][0, at // 16].long(), :, at % 16, 1] = (rise if size < 2.0 ** 12 else rise // 2 * 2)[:, None]
    expected = steps.chunk_attention(**case)
    actual = ops.paged_chunk_attention_native(**_to(case, gpu_device))
    _close(actual, expected, _bound({**case, "scale": 0.0}, expected))


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("heads,kv_heads,dim,tokens,before", CUT)
def test_scaled_scores_beyond_float32_in_cut_tiles(gpu_device, dtype, heads, kv_heads, dim, tokens, before):
    """16-bit scores are multiplied by the scale in the exponent's argument, after the maximum is taken off: three keys of 2^30
    among 2^29, times 1e30, share the row whether or not they lie in one part."""
    case = _chunk_case(dim + before + 4, dtype, heads, kv_heads, dim, 16, [(tokens, before)], scale=1e30)
    case["query"].zero_()[..., 0] = 2.0 ** 15
    key, table = case["key_pages"], case["page_table"][0].long()
    key.nan_to_num_().zero_()[..., 0] = 2.0 ** 14
    for j in (before // 8, before // 2, before - 1):
        key[table[j // 16], :, j % 16, 0] = 2.0 ** 15
    expected = steps.chunk_attention(**case)
    actual = ops.paged_chunk_attention_native(**_to(case, gpu_device))
    _close(actual, expected, _bound({**case, "scale": 0.0}, expected))


@pytest.mark.parametrize("vocab", [100, 128000])
def test_sampling_no_rows_gives_nothing(gpu_device, vocab):
    options = {name: torch.empty(0, device=gpu_device) for name in ("temperature", "top_p", "min_p")}
    tokens, probabilities = ops.logits_sample_native(torch.empty(0, vocab, device=gpu_device), torch.empty(0, device=gpu_device),
                                                     top_k=torch.empty(0, dtype=torch.int64, device=gpu_device), **options)
    assert tokens.shape == probabilities.shape == (0,) and tokens.dtype == torch.int64 and probabilities.dtype == torch.float32


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top_p,top_k", [(0.9, 0), (0.97, 90000), (1.0, 60000)])
def test_sampling_flat_rows(gpu_device, dtype, top_p, top_k):
    """More than 1024 tokens lie where the filters end, few of them equal: rows that one workgroup takes."""
    g = torch.Generator().manual_seed(31)
    logits = torch.randn(3, 152000, generator=g).to(dtype)
    options = {"uniforms": torch.rand(3, generator=g), "temperature": torch.tensor([1.0, 2.0, 0.9]), "top_p": torch.full((3,), top_p),
               "top_k": torch.tensor([top_k, top_k, 0]), "min_p": torch.tensor([0.0, 0.0, 1e-3])}
    _check_sample(logits, gpu_device, **options)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_layout_that_cuts_a_request_needs_its_positions(gpu_device, dtype):
    case = _chunk_case(41, dtype, 4, 2, 64, 16, [(5, 30), (40, 500), (3, 3)])
    slots, positions, counts = torch.arange(3), torch.tensor([30, 500, 3]), torch.tensor([5, 40, 3])
    offsets, *_ = ops.paged_step_layout_native(case["page_table"].to(gpu_device), *(t.to(gpu_device) for t in (slots, positions, counts)), 16, 33)
    assert offsets.tolist() == [0, 5, 33, 33]
    cut = {**case, "query": case["query"][:33].contiguous(), "offsets": offsets.cpu()}
    _check_chunk(cut, gpu_device, positions=positions)
    whole = steps.chunk_attention(**case)[:33]
    assert torch.equal(steps.chunk_attention(**cut, positions=positions), whole)
