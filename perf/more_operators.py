"""Timed cases of a served step in which prompts' chunks and single tokens run together, and of the sampling after it.

A case is a dict of plain values; ``kind`` names what one pass does:

* ``layout``: the step's tokens, packed one request after the other, get their places from the requests' slots, positions
  and counts (``paged_step_layout``).
* ``rows``: a layer's new K/V rows go to their rows of the pages (``paged_cache_write_rows``).
* ``chunk``: the packed tokens attend over their sequences' pages (``paged_chunk_attention``).
* ``sample``: a batch's next tokens from its logits, each row with its own temperature, top-k, top-p and min-p, and given
  random numbers (``logits_sample``): the tokens and the probabilities with which they were drawn.

Queries, keys and values are N(0, 1) (they follow an RMSNorm and a projection), logits N(0, 3).  Counts and lengths are a
function of the case alone; the seed draws their order and all values.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
    return [
        # A chat of this framework's model goes on: a short new message behind a few hundred tokens.
        {"name": "chunk_one_16", "kind": "chunk", "dtype": "float32", "query_heads": 9, "kv_heads": 3, "dim": 64,
         "page": 16, "requests": 1, "decoding": 0, "chunk": 16, "context": 884, "spare": 0, "window": 0, "sinks": 0},
        # Prompts of the same model in chunks: one at its start, others behind what was read before.
        {"name": "chunk_prompts_f32", "kind": "chunk", "dtype": "float32", "query_heads": 9, "kv_heads": 3, "dim": 64,
         "page": 16, "requests": 4, "decoding": 0, "chunk": 1024, "context": 7168, "spare": 0, "window": 0, "sinks": 0},
        # A served step in 16 bits: many sequences that decode, and two chunks of prompts, in a buffer of a fixed size.
        {"name": "chunk_mixed_bf16", "kind": "chunk", "dtype": "bfloat16", "query_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "requests": 50, "decoding": 48, "chunk": 1024, "context": 15360, "spare": 200, "window": 0,
         "sinks": 0},
        # A long document's last chunk: the most arithmetic.
        {"name": "chunk_long_bf16", "kind": "chunk", "dtype": "bfloat16", "query_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "requests": 1, "decoding": 0, "chunk": 4096, "context": 28672, "spare": 0, "window": 0, "sinks": 0},
        # One KV head, a head width and a page size that fill no tile evenly, a window behind long contexts.
        {"name": "chunk_window_f16", "kind": "chunk", "dtype": "float16", "query_heads": 8, "kv_heads": 1, "dim": 80,
         "page": 48, "requests": 24, "decoding": 8, "chunk": 333, "context": 20000, "spare": 11, "window": 2048,
         "sinks": 4},
        # Four chats, a few tokens each: the smallest step.
        {"name": "layout_4", "kind": "layout", "requests": 4, "decoding": 1, "chunk": 16, "context": 900, "page": 16,
         "slots": 16, "spare": 24},
        # A full step of a large server.
        {"name": "layout_1024", "kind": "layout", "requests": 1024, "decoding": 896, "chunk": 1024, "context": 30000,
         "page": 64, "slots": 1500, "spare": 1000},
        # The rows of a short message, this framework's heads.
        {"name": "rows_16", "kind": "rows", "dtype": "float32", "kv_heads": 3, "dim": 64, "page": 16, "tokens": 16,
         "pages": 256, "spare": 0},
        # A full step's rows in 16 bits.
        {"name": "rows_16384", "kind": "rows", "dtype": "bfloat16", "kv_heads": 8, "dim": 128, "page": 64,
         "tokens": 16384, "pages": 1024, "spare": 500},
        # The next token of one chat: this framework's vocabulary.
        {"name": "sample_one", "kind": "sample", "dtype": "float32", "batch": 1, "vocab": 49152, "filters": True},
        # A served batch over a large vocabulary, temperature alone.
        {"name": "sample_free_f32", "kind": "sample", "dtype": "float32", "batch": 32, "vocab": 128000, "filters": False},
        # A large batch in 16 bits (many equal logits), every row with its own mixture of filters.
        {"name": "sample_batch_bf16", "kind": "sample", "dtype": "bfloat16", "batch": 128, "vocab": 128000,
         "filters": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("chunk", "chunk", "chunk", "layout", "rows", "sample", "sample"))
    dtype = rng.choice(("float32", "bfloat16", "float16"))
    query_heads, kv_heads = rng.choice(((9, 3), (9, 3), (32, 8), (8, 1), (8, 8), (15, 5), (24, 2), (40, 8), (16, 16)))
    dim = rng.choice((32, 40, 64, 64, 72, 80, 96, 128, 128, 160, 256))
    page = rng.choice((8, 16, 16, 32, 48, 64, 100, 128))
    if kind == "chunk":
        requests = _log(rng, 1, 64)
        decoding = rng.choice((0, rng.randint(0, requests), requests))
        chunk = _log(rng, 1, 4096)
        context = rng.choice((0, _log(rng, 1, 28672), _log(rng, 256, 28672)))
        window = rng.choice((0, 0, _log(rng, 16, 4096)))
        case = {"kind": kind, "dtype": dtype, "query_heads": query_heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                "requests": requests, "decoding": decoding, "chunk": chunk, "context": context,
                "spare": rng.choice((0, rng.randint(1, 300))), "window": window,
                "sinks": rng.choice((0, 1, 4, 64)) if window else 0}
        most = listed()[3]
        limit = 4 * most["query_heads"] * most["dim"] * most["chunk"] * (most["chunk"] // 2 + most["context"])
        limit //= 8 if dtype == "float32" else 2
        while work({**case, "window": 0})["flops"] > limit or work(case)["bytes"] > 400_000_000:
            case["chunk"], case["context"] = -(-case["chunk"] * 3 // 4), case["context"] * 3 // 4
            if case["chunk"] <= 64 and case["requests"] > 1:
                case["requests"] = -(-case["requests"] // 2)
                case["decoding"] = min(case["decoding"], case["requests"])
        return case
    if kind == "layout":
        requests = _log(rng, 1, 1024)
        chunk = min(_log(rng, 1, 4096), 150_000 // requests + 1)
        return {"kind": kind, "requests": requests, "decoding": rng.randint(0, requests), "chunk": chunk,
                "context": rng.choice((0, _log(rng, 1, 30000))), "page": page, "slots": requests + rng.randint(0, 500),
                "spare": rng.choice((0, rng.randint(1, 1000)))}
    if kind == "rows":
        tokens = min(_log(rng, 1, 16384), 16384 * 8 * 128 * 2 // (kv_heads * dim * BYTES[dtype]))
        return {"kind": kind, "dtype": dtype, "kv_heads": kv_heads, "dim": dim, "page": page, "tokens": tokens,
                "pages": -(-tokens // page) + _log(rng, 1, 512), "spare": rng.choice((0, rng.randint(1, 300)))}
    batch = _log(rng, 1, 128)
    return {"kind": kind, "dtype": dtype, "batch": batch, "vocab": min(_log(rng, 1000, 200_000), 128 * 128_000 // batch),
            "filters": rng.random() < 0.7}


# ---------------------------------------------------------------------------
# Sizes that follow from a case.

def _spread(count, longest):
    """``count`` numbers from an eighth of ``longest`` up to it; the first is the longest."""
    low = longest // 8
    return [longest - (b * 7919) % (longest - low + 1) for b in range(count)]


def _requests(case):
    """(tokens, earlier keys) of every request: single tokens behind the chunks."""
    chunks = case["requests"] - case["decoding"]
    counts = [max(1, n) for n in _spread(chunks, case["chunk"])] + [1] * case["decoding"]
    return list(zip(counts, _spread(case["requests"], case["context"])))


def _tokens(case):
    return sum(count for count, _ in _requests(case)) + case["spare"]


def _visible(position, case):
    """Keys that the query at ``position`` sees."""
    seen, window = position + 1, case["window"]
    return seen if not window or seen <= window else window + min(case["sinks"], seen - window)


def work(case):
    kind = case["kind"]
    if kind == "layout":
        requests = _requests(case)
        entries = sum((before + count - 1) // case["page"] - before // case["page"] + 1 for count, before in requests)
        return {"bytes": 24 * len(requests) + 4 * entries + 8 * (len(requests) + 1) + 24 * _tokens(case), "flops": 0}
    size = BYTES[case["dtype"]]
    if kind == "rows":
        return {"bytes": 4 * case["tokens"] * case["kv_heads"] * case["dim"] * size + 8 * (case["tokens"] + case["spare"]),
                "flops": 0}
    if kind == "sample":
        rows = case["batch"]
        return {"bytes": size * rows * case["vocab"] + 32 * rows, "flops": 20 * rows * case["vocab"]}
    q, kv, dim = case["query_heads"], case["kv_heads"], case["dim"]
    pairs, keys, pages = 0, 0, 0
    for count, before in _requests(case):
        window, last = case["window"], before + count
        whole = min(count, max(0, window - before)) if window else count  # tokens that see all before them
        pairs += whole * before + whole * (whole + 1) // 2
        pairs += sum(_visible(p, case) for p in range(before + whole, last))
        oldest = max(0, before - window + 1) if window else 0
        seen = last - oldest + min(case["sinks"], oldest)
        keys += seen
        pages += -(-seen // case["page"])
    tokens = _tokens(case)
    return {"bytes": size * dim * (2 * kv * keys + q * (2 * tokens - case["spare"])) + 4 * pages + 24 * case["requests"],
            "flops": 4 * q * dim * pairs}


# ---------------------------------------------------------------------------
# Inputs.

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    kind = case["kind"]
    dtype = TYPES[case.get("dtype", "float32")]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)

    def order(count):
        return torch.randperm(count, generator=g, device=DEVICE)

    def uniform(count, low, high):
        return low + (high - low) * torch.rand(count, generator=g, device=DEVICE)

    s = {"case": case}
    if kind in ("layout", "chunk"):
        # The scheduler's lists: its program knows each request's count and how far its sequence has come.
        requests = _requests(case)
        s["spans"] = [requests[i] for i in torch.randperm(len(requests), generator=host).tolist()]
        counts, before = torch.tensor(s["spans"], device=DEVICE).T.contiguous()
        slot_count = case["slots"] if kind == "layout" else case["requests"] + 3
        s["slots"] = order(slot_count)[: len(requests)].contiguous()
        s["counts"], s["positions"] = counts, before
        s["lengths"] = torch.zeros(slot_count, dtype=torch.int64, device=DEVICE)
        s["lengths"][s["slots"]] = before + counts
        columns = max(-(-(c + b) // case["page"]) for c, b in s["spans"])
        needed = -(-s["lengths"] // case["page"])
        held = torch.arange(columns, device=DEVICE) < needed[:, None]
        pages = int(needed.sum()) + 7
        s["table"] = torch.full((slot_count, columns), -1, dtype=torch.int32, device=DEVICE)
        s["table"][held] = order(pages)[: pages - 7].to(torch.int32)
        s["tokens"] = _tokens(case)
    if kind == "chunk":
        q, kv, dim = case["query_heads"], case["kv_heads"], case["dim"]
        # The step's queries are a part of one projection's rows.
        s["query"] = normal(s["tokens"], q + 2 * kv, dim)[:, :q]
        s["key"], s["value"] = (normal(pages, kv, case["page"], dim) for _ in range(2))
        s["offsets"] = torch.nn.functional.pad(s["counts"].cumsum(0), (1, 0))
        s["scale"] = dim ** -0.5
    elif kind == "rows":
        tokens, both = case["tokens"] + case["spare"], 2 * case["kv_heads"]
        rows = normal(tokens, both, case["dim"])
        s["key"], s["value"] = rows[:, : case["kv_heads"]], rows[:, case["kv_heads"]:]
        # Runs of a page's rows, as chunks have them; what is behind the last token goes nowhere.
        pages = order(case["pages"])[: -(-case["tokens"] // case["page"])]
        s["rows"] = torch.full((tokens,), -1, dtype=torch.int64, device=DEVICE)
        s["rows"][: case["tokens"]] = (pages[:, None] * case["page"] + torch.arange(case["page"], device=DEVICE)
                                       ).flatten()[: case["tokens"]]
        shape = (case["pages"], case["kv_heads"], case["page"], case["dim"])
        s["key_pages"], s["value_pages"] = normal(*shape), normal(*shape)
    elif kind == "sample":
        rows = case["batch"]
        s["logits"] = normal(rows, case["vocab"]) * 3
        s["uniforms"] = uniform(rows, 0.0, 1.0)
        s["temperature"] = uniform(rows, 0.5, 1.3)
        s["top_k"] = s["top_p"] = s["min_p"] = None
        if case["filters"]:
            def some(share):
                return torch.rand(rows, generator=g, device=DEVICE) < share

            k = (10 ** (1 + 2 * torch.rand(rows, generator=g, device=DEVICE))).long()
            s["top_k"] = torch.where(some(0.5), k, 0)
            s["top_p"] = torch.where(some(0.7), uniform(rows, 0.7, 0.99), 1.0)
            s["min_p"] = torch.where(some(0.3), uniform(rows, 0.01, 0.1), 0.0)
            s["temperature"] = torch.where(some(0.1), 0.0, s["temperature"])  # these are greedy
    return s


# ---------------------------------------------------------------------------
# One pass.

def run(state):
    case = state["case"]
    return _PASSES[case["kind"]](state, case)


def _layout(s, case):
    if own:
        from flux_amd import ops

        return ops.paged_step_layout_native(s["table"], s["slots"], s["positions"], s["counts"], case["page"], s["tokens"])
    table, page = s["table"], case["page"]
    offsets = torch.nn.functional.pad(s["counts"].cumsum(0), (1, 0)).clamp(max=s["tokens"])
    token = torch.arange(s["tokens"], device=DEVICE)
    request = torch.searchsorted(offsets[1:], token, right=True)
    real = request < case["requests"]
    mine = request.clamp(max=case["requests"] - 1)
    position = s["positions"][mine] + token - offsets[mine]
    held = table[s["slots"][mine], (position // page).clamp(max=table.shape[1] - 1)].long()
    row = torch.where(held >= 0, held * page + position % page, -1)
    return [offsets, *(torch.where(real, t, -1) for t in (request, position, row))]


def _rows(s, case):
    if own:
        from flux_amd import ops

        ops.paged_cache_write_rows_native(s["key"], s["value"], s["key_pages"], s["value_pages"], s["rows"])
        return [s["key_pages"], s["value_pages"]]
    real = s["rows"] >= 0
    page, row = s["rows"][real] // case["page"], s["rows"][real] % case["page"]
    s["key_pages"][page, :, row] = s["key"][real]
    s["value_pages"][page, :, row] = s["value"][real]
    return [s["key_pages"], s["value_pages"]]


def _chunk(s, case):
    if own:
        from flux_amd import ops

        return ops.paged_chunk_attention_native(s["query"], s["key"], s["value"], s["table"], s["lengths"], s["offsets"],
                                                s["scale"], case["window"], case["sinks"], s["slots"])
    q, kv, dim, page = (case[k] for k in ("query_heads", "kv_heads", "dim", "page"))
    out = torch.zeros(s["tokens"], q, dim, dtype=s["query"].dtype, device=DEVICE)
    first = 0
    for i, (count, before) in enumerate(s["spans"]):
        keys = before + count
        pages = s["table"][s["slots"][i], : -(-keys // page)].long()
        position = torch.arange(before, keys, device=DEVICE)[:, None]
        at = torch.arange(keys, device=DEVICE)
        hidden = at > position
        if case["window"]:
            hidden |= (at <= position - case["window"]) & (at >= case["sinks"])
        group = q // kv
        for h in range(kv):
            key, value = (t[pages, h].reshape(-1, dim)[:keys].float() for t in (s["key"], s["value"]))
            query = s["query"][first : first + count, h * group : (h + 1) * group].float()
            score = torch.matmul(query.reshape(-1, dim), key.T).mul_(s["scale"]).view(count, group, keys)
            score.masked_fill_(hidden[:, None], -math.inf)
            score -= score.amax(-1, keepdim=True)
            weight = score.exp_()
            mean = torch.matmul(weight.view(-1, keys), value).view(count, group, dim) / weight.sum(-1, keepdim=True)
            out[first : first + count, h * group : (h + 1) * group] = mean.to(out.dtype)
        first += count
    return out


def _sample(s, case):
    if own:
        from flux_amd import ops

        return ops.logits_sample_native(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    # In 64 bits: a sum of so many weights in 32 would move the borders between the tokens.
    x, vocab = s["logits"].double(), case["vocab"]
    top = x.amax(1, keepdim=True)
    at = torch.arange(vocab, device=DEVICE)
    greedy = torch.where(x == top, at, vocab).amin(1)
    temperature = s["temperature"].double()[:, None]
    weight = torch.exp((x - top) / torch.where(temperature > 0, temperature, 1.0))
    if case["filters"]:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        mass = weight.gather(1, order)
        k = s["top_k"][:, None]
        kept = (at < k) | (k <= 0)
        mass = torch.where(kept, mass, 0.0)
        before = mass.cumsum(1) - mass
        p = s["top_p"].double()[:, None]
        kept &= (p >= 1) | (before < p * mass.sum(1, keepdim=True)) | (at == 0)
        kept &= mass >= s["min_p"].double()[:, None].clamp(max=1.0)
        weight = torch.zeros_like(weight).scatter_(1, order, torch.where(kept, mass, 0.0))
    reached = weight.cumsum(1)
    target = s["uniforms"].double()[:, None] * reached[:, -1:]
    token = (reached <= target).sum(1)
    probability = weight.gather(1, token[:, None])[:, 0] / reached[:, -1]
    drawn = s["temperature"] > 0
    return [torch.where(drawn, token, greedy), torch.where(drawn, probability, 1.0).float()]


_PASSES = {"layout": _layout, "rows": _rows, "chunk": _chunk, "sample": _sample}


# ---------------------------------------------------------------------------
# The definitions, in 64 bits where numbers are computed, one request, head or row at a time.

def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s, case)


def _exact_layout(s, case):
    table, slots = s["table"].tolist(), s["slots"].tolist()
    offsets, request, position, row = [0], [], [], []
    for i, (count, before) in enumerate(s["spans"]):
        offsets.append(offsets[-1] + count)
        request += [i] * count
        position += range(before, before + count)
        row += [table[slots[i]][p // case["page"]] * case["page"] + p % case["page"] for p in range(before, before + count)]
    behind = [-1] * case["spare"]
    return [torch.tensor(values) for values in (offsets, request + behind, position + behind, row + behind)]


def _exact_rows(s, case):
    for pages, new in ((s["key_pages"], s["key"]), (s["value_pages"], s["value"])):
        flat = pages.transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
        flat.index_copy_(0, s["rows"][: case["tokens"]], new[: case["tokens"]])
        pages.copy_(flat.view(case["pages"], case["page"], case["kv_heads"], case["dim"]).transpose(1, 2))
    return [s["key_pages"], s["value_pages"]]


def _exact_chunk(s, case):
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEVICE)
    group, page = case["query_heads"] // case["kv_heads"], case["page"]
    offsets = s["offsets"].tolist()
    for i, n in enumerate(s["lengths"][s["slots"]].tolist()):
        low, high = offsets[i], offsets[i + 1]
        for start in range(low, high, 512):
            rows = torch.arange(start, min(start + 512, high), device=DEVICE)
            p = (n - high + rows)[:, None]
            j = torch.arange(n, device=DEVICE)
            if case["window"]:
                j = j[(j > int(p.min()) - case["window"]) | (j < case["sinks"])]
            seen = j <= p
            if case["window"]:
                seen &= (j > p - case["window"]) | (j < case["sinks"])
            held = s["table"][s["slots"][i], j // page].long()
            for h in range(case["kv_heads"]):
                key, value = (t[held, h, j % page].double() for t in (s["key"], s["value"]))
                for of in range(h * group, (h + 1) * group):
                    score = (s["query"][rows, of].double() @ key.T) * s["scale"]
                    out[rows, of] = torch.softmax(torch.where(seen, score, -math.inf), dim=1) @ value
    return out


def _exact_sample(s, case):
    logits = s["logits"].double().cpu().numpy()
    rows = {k: None if s[k] is None else s[k].double().cpu().numpy()
            for k in ("uniforms", "temperature", "top_k", "top_p", "min_p")}
    tokens, probabilities = [], []
    for b, x in enumerate(logits):
        best = int(np.argmax(x))  # numpy's is the first of the largest
        if not rows["temperature"][b] > 0:
            tokens.append(best)
            probabilities.append(1.0)
            continue
        weight = np.exp((x - x[best]) / rows["temperature"][b])
        kept = np.arange(len(x))
        if case["filters"]:
            kept = np.lexsort((kept, -x))
            if rows["top_k"][b] > 0:
                kept = kept[: int(rows["top_k"][b])]
            if rows["top_p"][b] < 1:
                reached = np.cumsum(weight[kept])
                kept = kept[: 1 + np.count_nonzero(reached[:-1] < rows["top_p"][b] * reached[-1])]
            kept = np.sort(kept[weight[kept] >= min(rows["min_p"][b], 1.0)])
        reached = np.cumsum(weight[kept])
        tokens.append(int(kept[np.searchsorted(reached, rows["uniforms"][b] * reached[-1], side="right")]))
        probabilities.append(weight[tokens[-1]] / reached[-1])
    return [torch.tensor(tokens), torch.tensor(probabilities, dtype=torch.float64)]


_EXACT = {"layout": _exact_layout, "rows": _exact_rows, "chunk": _exact_chunk, "sample": _exact_sample}
