"""Timed cases of the serving operators: attention over a paged K/V cache, windowed attention, pages, logits.

A case is a dict of plain values; ``kind`` names what one pass does, as a program that serves several sequences does it:

* ``paged``: one new token of every sequence of a batch attends over its pages (``paged_decode_attention``).
* ``window``: the queries of a prompt, of a chunk of it or of single tokens attend over contiguous K/V with a sliding
  window and sink tokens (``window_attention``).
* ``admit``: finished sequences give their pages back, new prompts get pages, and a layer writes their K/V rows
  (``paged_cache_free``, ``paged_cache_reserve``, ``paged_cache_write``).
* ``fork``: branches of shared prompts are dropped and branched again (``paged_cache_free``, ``paged_cache_fork``).
* ``compact``: the pages in use move to the front of the pool (``paged_cache_compact``).
* ``copy``: pages of all layers are copied inside the pool (``paged_cache_copy``).
* ``logits``: penalties, bias and grammar mask on a batch's logits, and the greedy tokens (``logits_process``).

Queries, keys and values are N(0, 1) (they follow an RMSNorm and a projection), logits N(0, 3).  Sequence lengths and
the numbers of pages that move are a function of the case alone; the seed draws their order and all values.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
ATTENTION = ("query_heads", "kv_heads", "dim")


def listed():
    return [
        # One chat of this framework's model, its cache in pages: the smallest step, where latency counts.
        {"name": "paged_one_900", "kind": "paged", "dtype": "float32", "batch": 1, "query_heads": 9, "kv_heads": 3,
         "dim": 64, "page": 16, "longest": 900, "window": 0, "sinks": 0},
        # The same heads for a served batch of ragged contexts up to the benchmark's.
        {"name": "paged_ragged_8192", "kind": "paged", "dtype": "float32", "batch": 24, "query_heads": 9,
         "kv_heads": 3, "dim": 64, "page": 16, "longest": 8192, "window": 0, "sinks": 0},
        # A large batch of long contexts in 16 bits, wider heads: the largest cache read.
        {"name": "paged_long_bf16", "kind": "paged", "dtype": "bfloat16", "batch": 48, "query_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "longest": 16384, "window": 0, "sinks": 0},
        # One KV head, a head width and a page size that fill no tile evenly, a window behind long contexts.
        {"name": "paged_window_f16", "kind": "paged", "dtype": "float16", "batch": 64, "query_heads": 8, "kv_heads": 1,
         "dim": 80, "page": 48, "longest": 20000, "window": 2048, "sinks": 4},
        # A document's prompt through a layer of this framework's model with a window.
        {"name": "window_prompt_4096", "kind": "window", "dtype": "float32", "batch": 1, "query_heads": 9,
         "kv_heads": 3, "dim": 64, "queries": 4096, "keys": 4096, "window": 1024, "sinks": 4, "padded": True},
        # A padded batch of prompts in 16 bits, wider heads: the most arithmetic.
        {"name": "window_batch_bf16", "kind": "window", "dtype": "bfloat16", "batch": 4, "query_heads": 32,
         "kv_heads": 8, "dim": 128, "queries": 4096, "keys": 4096, "window": 1024, "sinks": 16, "padded": True},
        # New prompts of a few hundred tokens take over the slots of finished sequences.
        {"name": "admit_16", "kind": "admit", "dtype": "float32", "slots": 16, "longest": 1000, "kv_heads": 3, "dim": 64,
         "page": 16, "pages": 2048},
        # Eight shared prompts, eight branches each: all layers' last pages are copied.
        {"name": "fork_64", "kind": "fork", "dtype": "float32", "parents": 8, "branches": 8, "longest": 700,
         "layers": 30, "kv_heads": 3, "dim": 64, "page": 16, "pages": 512},
        # A pool after many sequences came and went: a quarter of it moves.
        {"name": "compact_512", "kind": "compact", "dtype": "bfloat16", "pages": 2048, "used": 1024, "moved": 512,
         "layers": 8, "kv_heads": 8, "dim": 128, "page": 16, "slots": 64},
        # A scheduler duplicates a few pages before sequences that share them write on.
        {"name": "copy_40", "kind": "copy", "dtype": "float32", "pages": 512, "copies": 40, "layers": 30, "kv_heads": 3,
         "dim": 64, "page": 16},
        # The next token of one chat: this framework's vocabulary, its whole history.
        {"name": "logits_one", "kind": "logits", "dtype": "float32", "batch": 1, "vocab": 49152, "history": 700},
        # A served batch over a large vocabulary in 16 bits, long histories.
        {"name": "logits_batch_bf16", "kind": "logits", "dtype": "bfloat16", "batch": 128, "vocab": 128000,
         "history": 4096},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("paged", "paged", "window", "window", "admit", "fork", "compact", "copy", "logits", "logits"))
    dtype = rng.choice(("float32", "float32", "bfloat16", "float16"))
    query_heads, kv_heads = rng.choice(((9, 3), (9, 3), (32, 8), (8, 1), (8, 8), (15, 5), (24, 2), (40, 8), (16, 16)))
    dim = rng.choice((32, 40, 64, 64, 72, 80, 96, 128, 128, 160, 256))
    page = rng.choice((8, 16, 16, 32, 48, 64, 100, 128))
    pool = {"kv_heads": kv_heads, "dim": dim, "page": page}
    if kind == "paged":
        batch = _log(rng, 1, 128)
        most = 40 * 16384 * 8 * 128 * 2 // (batch * kv_heads * dim * BYTES[dtype])
        longest = min(_log(rng, 16, 32768), most, 32 * 20000 // batch + 16)
        window = rng.choice((0, 0, _log(rng, 16, 8192)))
        return {"kind": kind, "dtype": dtype, "batch": batch, "query_heads": query_heads, **pool, "longest": longest,
                "window": window, "sinks": rng.choice((0, 1, 4, 64)) if window else 0}
    if kind == "window":
        batch = _log(rng, 1, 16)
        queries = rng.choice((1, _log(rng, 2, 8192), _log(rng, 64, 8192)))
        keys = max(queries, rng.choice((queries, _log(rng, 16, 16384))))
        most = 4 * 32 * 4096 * 4096 // (batch * query_heads)
        keys = min(keys, max(64, most // queries))
        queries = min(queries, keys, math.isqrt(most))
        keys = min(keys, most // queries)
        if queries > 1 and dim > 128:
            dim = 128
        widest = 4 * 32 * 4096 * 500 * 128 // (batch * query_heads * queries * dim)
        return {"kind": kind, "dtype": dtype, "batch": batch, "query_heads": query_heads, "kv_heads": kv_heads,
                "dim": dim, "queries": queries, "keys": keys, "window": min(_log(rng, 16, 2048), widest),
                "sinks": rng.choice((0, 1, 4, 64)), "padded": queries == keys}
    if kind == "admit":
        slots, longest = _log(rng, 1, 64), _log(rng, 4, 2000)
        pages = slots * -(-longest // page) + _log(rng, 64, 4096)
        return {"kind": kind, "dtype": dtype, "slots": slots, "longest": longest, **pool, "pages": pages}
    layers = rng.randint(1, 30)
    row = kv_heads * dim * BYTES[dtype]
    most = 400_000_000 // (page * row)  # pages of one layer that a pool of 400 MB holds
    if kind == "fork":
        parents, branches, longest = _log(rng, 1, 16), _log(rng, 1, 16), _log(rng, 2, 1500)
        pages = parents * (-(-longest // page) + branches) + 8
        return {"kind": kind, "dtype": dtype, "parents": parents, "branches": branches, "longest": longest,
                "layers": max(1, min(layers, most // pages)), **pool, "pages": pages}
    pages = min(_log(rng, 32, 4096), max(32, most // layers))
    layers = max(1, min(layers, most // pages))
    if kind == "copy":
        return {"kind": kind, "dtype": dtype, "pages": pages, "copies": _log(rng, 1, pages // 2), "layers": layers, **pool}
    if kind == "compact":
        used = rng.randint(2, pages - 2)
        return {"kind": kind, "dtype": dtype, "pages": pages, "used": used,
                "moved": rng.randint(1, min(used, pages - used)), "layers": layers, **pool, "slots": _log(rng, 1, 128)}
    batch = _log(rng, 1, 256)
    vocab = min(_log(rng, 1000, 200_000), 128 * 128_000 // batch)
    return {"kind": kind, "dtype": dtype, "batch": batch, "vocab": vocab, "history": min(_log(rng, 1, 8192), 4096 * 128 // batch)}


# ---------------------------------------------------------------------------
# Sizes that follow from a case.

def _lengths(count, longest):
    """``count`` lengths from an eighth of ``longest`` up to it; the first is the longest."""
    low = max(1, longest // 8)
    return [longest - (b * 7919) % (longest - low + 1) for b in range(count)]


def _starts(case):
    return [0 if case["padded"] else n - case["queries"] for n in _window_lengths(case)]


def _window_lengths(case):
    if case["padded"]:
        return _lengths(case["batch"], case["keys"])
    return [max(n, case["queries"]) for n in _lengths(case["batch"], case["keys"])]


def _visible(position, case):
    """Keys that the query at ``position`` sees."""
    seen, window = position + 1, case["window"]
    return seen if not window or seen <= window else window + min(case["sinks"], seen - window)


def work(case):
    size = BYTES[case["dtype"]]
    kind = case["kind"]
    if kind == "paged":
        q, kv, dim = (case[k] for k in ATTENTION)
        seen = [_visible(n - 1, case) for n in _lengths(case["batch"], case["longest"])]
        pages = sum(-(-n // case["page"]) for n in seen)
        return {"bytes": size * dim * (2 * kv * sum(seen) + 2 * q * case["batch"]) + 4 * pages + 8 * case["batch"],
                "flops": 4 * q * dim * sum(seen)}
    if kind == "window":
        q, kv, dim = (case[k] for k in ATTENTION)
        pairs, keys = 0, 0
        for n, first in zip(_window_lengths(case), _starts(case)):
            last = min(first + case["queries"], n)
            pairs += sum(_visible(p, case) for p in range(first, last))
            oldest = max(0, first - case["window"] + 1)
            keys += last - oldest + min(case["sinks"], oldest)
        out = case["batch"] * case["queries"]
        return {"bytes": size * dim * (2 * kv * keys + 2 * q * out), "flops": 4 * q * dim * pairs}
    if kind == "logits":
        rows, vocab = case["batch"], case["vocab"]
        return {"bytes": 2 * size * rows * vocab + 4 * vocab + 4 * rows * (-(-vocab // 32)) +
                8 * sum(_lengths(rows, case["history"])) + 20 * rows, "flops": 6 * rows * vocab}
    row = 2 * case["kv_heads"] * case["dim"] * size  # K and V of one token
    if kind == "admit":
        lengths = _lengths(case["slots"], case["longest"])
        pages = sum(-(-n // case["page"]) for n in lengths)
        return {"bytes": 2 * row * sum(lengths) + 24 * pages + 4 * case["pages"], "flops": 0}
    if kind == "fork":
        lengths = _lengths(case["parents"], case["longest"])
        rows = case["branches"] * sum(n % case["page"] for n in lengths)
        pages = case["branches"] * sum(-(-n // case["page"]) for n in lengths)
        return {"bytes": 2 * row * case["layers"] * rows + 24 * pages + 4 * case["pages"], "flops": 0}
    moved = case["moved"] if kind == "compact" else case["copies"]
    return {"bytes": 2 * row * case["layers"] * case["page"] * moved + 8 * case["pages"], "flops": 0}


# ---------------------------------------------------------------------------
# Inputs.

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, kind = TYPES[case["dtype"]], case["kind"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)

    def order(count):
        return torch.randperm(count, generator=g, device=DEVICE)

    def shuffled(values, dtype=torch.int64):
        return torch.tensor(values, dtype=dtype, device=DEVICE)[order(len(values))]

    s = {"case": case}
    if kind in ("paged", "window"):
        q, kv, dim = (case[k] for k in ATTENTION)
        s["scale"] = dim ** -0.5
    if kind == "paged":
        s["lengths"] = shuffled(_lengths(case["batch"], case["longest"]))
        columns = -(-case["longest"] // case["page"])
        needed = -(-s["lengths"] // case["page"])
        held = torch.arange(columns, device=DEVICE) < needed[:, None]
        pages = int(needed.sum()) + 7
        table = torch.full((case["batch"], columns), -1, dtype=torch.int32, device=DEVICE)
        table[held] = order(pages)[: pages - 7].to(torch.int32)
        s |= {"table": table, "query": normal(case["batch"], q, 1, dim),
              "key": normal(pages, kv, case["page"], dim), "value": normal(pages, kv, case["page"], dim)}
    elif kind == "window":
        # A prompt's q, k and v are views of one projection's rows.
        both = torch.tensor([_window_lengths(case), _starts(case)], device=DEVICE)[:, order(case["batch"])]
        s["lengths"], s["starts"] = both.contiguous()
        s["query"] = normal(case["batch"], case["queries"], q, dim).transpose(1, 2)
        s["key"], s["value"] = (normal(case["batch"], case["keys"], kv, dim).transpose(1, 2) for _ in range(2))
    elif kind == "logits":
        rows, vocab = case["batch"], case["vocab"]
        s["logits"] = normal(rows, vocab) * 3
        # Half of a history repeats a few tokens.
        ids = torch.randint(0, vocab, (rows, case["history"]), generator=g, device=DEVICE)
        often = torch.rand(ids.shape, generator=g, device=DEVICE) < 0.5
        s["history"] = torch.where(often, ids % min(vocab, 50), ids)
        s["history_lengths"] = shuffled(_lengths(rows, case["history"]))
        s["repetition"], s["frequency"], s["presence"] = (
            low + (high - low) * torch.rand(rows, generator=g, device=DEVICE)
            for low, high in ((1.0, 1.5), (0.0, 0.5), (0.0, 1.0)))
        s["bias"] = torch.randn(1, vocab, generator=g, device=DEVICE)
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g, device=DEVICE,
                                     dtype=torch.int64).to(torch.int32)
    elif kind == "admit":
        shape = (case["pages"], case["kv_heads"], case["page"], case["dim"])
        columns = -(-case["longest"] // case["page"])
        s |= {"key_pages": normal(*shape), "value_pages": normal(*shape),
              "table": torch.full((case["slots"], columns), -1, dtype=torch.int32, device=DEVICE),
              "lengths": torch.zeros(case["slots"], dtype=torch.int64, device=DEVICE),
              "slots": order(case["slots"]), "counts": shuffled(_lengths(case["slots"], case["longest"]))}
        # Pages that other sequences hold, as many as leave room.
        spare = case["pages"] - case["slots"] * columns
        s["refcounts"] = torch.zeros(case["pages"], dtype=torch.int32, device=DEVICE)
        s["refcounts"][order(case["pages"])[: spare // 2]] = 1
        s["key"], s["value"] = (normal(case["slots"], case["longest"], case["kv_heads"], case["dim"]).transpose(1, 2)
                                for _ in range(2))
    else:
        shape = (case["layers"], case["pages"], case["kv_heads"], case["page"], case["dim"])
        s |= {"key_pages": normal(*shape), "value_pages": normal(*shape)}
    if kind == "fork":
        lengths = shuffled(_lengths(case["parents"], case["longest"]))
        slots = case["parents"] * (1 + case["branches"])
        columns = -(-case["longest"] // case["page"])
        needed = -(-lengths // case["page"])
        held = torch.arange(columns, device=DEVICE) < needed[:, None]
        used = order(case["pages"])[: int(needed.sum())]
        s["table"] = torch.full((slots, columns), -1, dtype=torch.int32, device=DEVICE)
        rows = torch.full((case["parents"], columns), -1, dtype=torch.int32, device=DEVICE)
        rows[held] = used.to(torch.int32)
        where = order(slots)
        s["table"][where[: case["parents"]]] = rows
        s["lengths"] = torch.zeros(slots, dtype=torch.int64, device=DEVICE)
        s["lengths"][where[: case["parents"]]] = lengths
        s["refcounts"] = torch.zeros(case["pages"], dtype=torch.int32, device=DEVICE)
        s["refcounts"][used] = 1
        s["parents"] = where[: case["parents"]].repeat(case["branches"])
        s["children"] = where[case["parents"]:].contiguous()
    elif kind == "compact":
        low, high = order(case["used"]), case["used"] + order(case["pages"] - case["used"])
        used = torch.cat((low[case["moved"]:], high[: case["moved"]]))
        used = used[order(case["used"])]
        # Sequences of one length, two of them sharing a first page now and then.
        columns = -(-case["used"] // case["slots"])
        flat = torch.full((case["slots"] * columns,), -1, dtype=torch.int32, device=DEVICE)
        flat[: case["used"]] = used.to(torch.int32)
        s["table"] = flat.view(case["slots"], columns)
        s["refcounts"] = torch.zeros(case["pages"], dtype=torch.int32, device=DEVICE)
        s["refcounts"][used] = 1
        shared = torch.rand(case["slots"], generator=g, device=DEVICE) < 0.2
        spread = torch.cat((s["table"], torch.where(shared, s["table"][:1, 0], -1)[:, None]), dim=1)
        s["refcounts"][used[0]] += shared.sum()
        s["table"] = spread.contiguous()
    elif kind == "copy":
        both = order(case["pages"])
        s["source"], s["target"] = both[: case["copies"]], both[case["copies"]: 2 * case["copies"]]
    return s


# ---------------------------------------------------------------------------
# One pass.

def run(state):
    case = state["case"]
    return _PASSES[case["kind"]](state, case)


def _paged(s, case):
    if own:
        from flux_amd import ops

        return ops.paged_decode_attention_native(s["query"], s["key"], s["value"], s["table"], s["lengths"], s["scale"],
                                                 case["window"], case["sinks"])
    batch, columns = s["table"].shape
    q, kv, dim = (case[k] for k in ATTENTION)
    keys = columns * case["page"]
    pages = s["table"].clamp(min=0).long()
    key, value = (t[pages].float().permute(0, 2, 1, 3, 4).reshape(batch, kv, keys, dim) for t in (s["key"], s["value"]))
    at = torch.arange(keys, device=DEVICE)
    length = s["lengths"][:, None]
    seen = at < length
    if case["window"]:
        seen &= (at >= length - case["window"]) | (at < case["sinks"])
    score = torch.matmul(s["query"].float().reshape(batch, kv, q // kv, dim), key.transpose(2, 3)) * s["scale"]
    return _weighted(score, seen[:, None, None], value).reshape(batch, q, 1, dim).to(s["query"].dtype)


def _weighted(score, seen, value):
    """Softmax over the seen keys, times the values; nothing seen gives zeros."""
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    return torch.matmul(weight, value) / torch.where(total == 0, 1.0, total)


def _window(s, case):
    if own:
        from flux_amd import ops

        return ops.window_attention_native(s["query"], s["key"], s["value"], s["scale"], case["window"], case["sinks"],
                                           s["lengths"], s["starts"])
    q, kv, dim = (case[k] for k in ATTENTION)
    batch, rows, keys = case["batch"], case["queries"], case["keys"]
    key, value = (t.float().unsqueeze(2) for t in (s["key"], s["value"]))
    query = s["query"].float().reshape(batch, kv, q // kv, rows, dim)
    score = torch.matmul(query, key.transpose(3, 4)) * s["scale"]
    at = torch.arange(keys, device=DEVICE)
    position = (s["starts"][:, None] + torch.arange(rows, device=DEVICE))[:, :, None]
    seen = (at <= position) & (at < s["lengths"][:, None, None]) & (position < s["lengths"][:, None, None])
    seen &= (at > position - case["window"]) | (at < case["sinks"])
    out = _weighted(score, seen[:, None, None], value)
    return out.reshape(batch, q, rows, dim).to(s["query"].dtype)


def _admit(s, case):
    pools = s["key_pages"], s["value_pages"]
    state = s["table"], s["lengths"], s["refcounts"]
    if own:
        from flux_amd import ops

        ops.paged_cache_free_native(*state, s["slots"])
        positions, status = ops.paged_cache_reserve_native(*state, case["page"], s["slots"], s["counts"])
        ops.paged_cache_write_native(s["key"], s["value"], *pools, s["table"], s["slots"], positions, s["counts"])
        return [*pools, *state, positions, status]
    _release(*state, s["slots"])
    table, lengths, refcounts = state
    slots, counts, page = s["slots"], s["counts"], case["page"]
    positions = lengths[slots]
    after = positions + counts
    first = torch.arange(table.shape[1], device=DEVICE) * page
    needed = (first < after[:, None]) & (first + page > positions[:, None]) & (table[slots] < 0)
    free = torch.argsort((refcounts > 0).to(torch.int32), stable=True)
    got = free[(needed.flatten().cumsum(0) - 1).clamp(min=0)].view_as(needed)
    table[slots] = torch.where(needed, got.to(torch.int32), table[slots])
    refcounts[got[needed]] = 1
    lengths[slots] = after
    at = positions[:, None] + torch.arange(case["longest"], device=DEVICE)
    new = at < after[:, None]
    target = torch.gather(table[slots], 1, (at // page).clamp(max=table.shape[1] - 1)).long()[new]
    rows = (at % page)[new]
    pools[0][target, :, rows] = s["key"].transpose(1, 2)[new]
    pools[1][target, :, rows] = s["value"].transpose(1, 2)[new]
    return [*pools, *state, positions, torch.zeros_like(slots, dtype=torch.int32)]


def _release(table, lengths, refcounts, slots):
    rows = table[slots].flatten()
    refcounts.scatter_add_(0, rows.clamp(min=0).long(), -(rows >= 0).to(torch.int32))
    table[slots] = -1
    lengths[slots] = 0


def _fork(s, case):
    pools = s["key_pages"], s["value_pages"]
    state = s["table"], s["lengths"], s["refcounts"]
    if own:
        from flux_amd import ops

        ops.paged_cache_free_native(*state, s["children"])
        status = ops.paged_cache_fork_native(*pools, *state, s["parents"], s["children"])
        return [*pools, *state, status]
    _release(*state, s["children"])
    table, lengths, refcounts = state
    parents, children, page = s["parents"], s["children"], case["page"]
    length = lengths[parents]
    rest = length % page
    needed = rest > 0
    free = torch.argsort((refcounts > 0).to(torch.int32), stable=True)
    got = free[(needed.cumsum(0) - 1).clamp(min=0)]
    column = torch.arange(table.shape[1], device=DEVICE)
    full = (length // page)[:, None]
    rows = torch.where(column < full, table[parents], -1)
    refcounts.scatter_add_(0, rows.flatten().clamp(min=0).long(), (rows.flatten() >= 0).to(torch.int32))
    refcounts[got[needed]] = 1
    table[children] = torch.where((column == full) & needed[:, None], got[:, None].to(torch.int32), rows)
    lengths[children] = length
    last = torch.gather(table[parents], 1, (length // page).clamp(max=table.shape[1] - 1)[:, None])[:, 0].long()[needed]
    got, kept = got[needed], (torch.arange(page, device=DEVICE) < rest[needed][:, None])[None, :, None, :, None]
    pools[0][:, got] = torch.where(kept, pools[0][:, last], pools[0][:, got])
    pools[1][:, got] = torch.where(kept, pools[1][:, last], pools[1][:, got])
    return [*pools, *state, torch.zeros_like(parents, dtype=torch.int32)]


def _compact(s, case):
    # The tables are copied so that every pass finds the scattered pool: the moved pages' old rows stay as they are.
    pools = s["key_pages"], s["value_pages"]
    table, refcounts = s["table"].clone(), s["refcounts"].clone()
    if own:
        from flux_amd import ops

        page_map, used = ops.paged_cache_compact_native(*pools, table, refcounts)
        return [*pools, table, refcounts, page_map, used]
    held = refcounts > 0
    used = held.sum()
    at = torch.arange(case["pages"], device=DEVICE)
    source, target = (held & (at >= used)).nonzero()[:, 0], (~held & (at < used)).nonzero()[:, 0]
    page_map = torch.where(held, at, -1).to(torch.int32)
    page_map[source] = target.to(torch.int32)
    pools[0][:, target] = pools[0][:, source]
    pools[1][:, target] = pools[1][:, source]
    refcounts[target] = refcounts[source]
    refcounts[source] = 0
    table = torch.where(table >= 0, page_map[table.clamp(min=0).long()], -1)
    return [*pools, table, refcounts, page_map, used]


def _copy(s, case):
    pools = s["key_pages"], s["value_pages"]
    if own:
        from flux_amd import ops

        return [*pools, ops.paged_cache_copy_native(*pools, s["source"], s["target"])]
    pools[0][:, s["target"]] = pools[0][:, s["source"]]
    pools[1][:, s["target"]] = pools[1][:, s["source"]]
    return [*pools, torch.zeros_like(s["source"], dtype=torch.int32)]


def _logits(s, case):
    if own:
        from flux_amd import ops

        return ops.logits_process_native(s["logits"], s["history"], s["history_lengths"], s["repetition"],
                                         s["frequency"], s["presence"], s["bias"], s["allowed"])
    rows, vocab = s["logits"].shape
    inside = torch.arange(case["history"], device=DEVICE) < s["history_lengths"][:, None]
    count = torch.zeros(rows, vocab, device=DEVICE)
    count.scatter_add_(1, s["history"], inside.float())
    repetition, frequency, presence = (s[k][:, None] for k in ("repetition", "frequency", "presence"))
    x = s["logits"].float()
    x = torch.where(count > 0, torch.where(x > 0, x / repetition, x * repetition), x)
    x = x - frequency * count
    x = x - presence * (count > 0).float()
    x = x + s["bias"]
    at = torch.arange(vocab, device=DEVICE)
    bit = (s["allowed"][:, at // 32] >> (at % 32).to(torch.int32)) & 1
    x = torch.where(bit == 1, x, -math.inf).to(s["logits"].dtype)
    return [x, torch.where(x == x.amax(1, keepdim=True), at, vocab).amin(1)]


_PASSES = {"paged": _paged, "window": _window, "admit": _admit, "fork": _fork, "compact": _compact, "copy": _copy,
           "logits": _logits}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, one sequence, head or page at a time.

def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s, case)


def _attend_64(query, key, value, seen, scale):
    """query [rows, D], key and value [n, D], seen [rows, n] of one head."""
    score = (query.double() @ key.double().T) * scale
    weight = torch.softmax(torch.where(seen, score, -math.inf), dim=1)
    return torch.nan_to_num(weight, nan=0.0) @ value.double()


def _exact_paged(s, case):
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEVICE)
    group = case["query_heads"] // case["kv_heads"]
    for b, n in enumerate(s["lengths"].tolist()):
        at = torch.arange(n, device=DEVICE)
        if case["window"]:
            at = at[(at >= n - case["window"]) | (at < case["sinks"])]
        pages, rows = s["table"][b, at // case["page"]].long(), at % case["page"]
        for h in range(case["kv_heads"]):
            mine = slice(h * group, (h + 1) * group)
            everything = torch.ones(group, len(at), dtype=torch.bool, device=DEVICE)
            out[b, mine, 0] = _attend_64(s["query"][b, mine, 0], s["key"][pages, h, rows], s["value"][pages, h, rows],
                                         everything, s["scale"])
    return out


def _exact_window(s, case):
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEVICE)
    group = case["query_heads"] // case["kv_heads"]
    step = 1024
    for b, (n, first) in enumerate(zip(s["lengths"].tolist(), s["starts"].tolist())):
        for low in range(0, min(case["queries"], n - first), step):
            rows = slice(low, min(low + step, case["queries"], n - first))
            p = first + torch.arange(rows.start, rows.stop, device=DEVICE)[:, None]
            j = torch.arange(n, device=DEVICE)
            seen = (j <= p) & ((j > p - case["window"]) | (j < case["sinks"]))
            for h in range(case["query_heads"]):
                out[b, h, rows] = _attend_64(s["query"][b, h, rows], s["key"][b, h // group, :n],
                                             s["value"][b, h // group, :n], seen, s["scale"])
    return out


def _exact_logits(s, case):
    out = torch.empty(s["logits"].shape, dtype=torch.float64, device=DEVICE)
    bits = torch.arange(32, device=DEVICE)
    for b, n in enumerate(s["history_lengths"].tolist()):
        count = torch.bincount(s["history"][b, :n], minlength=case["vocab"]).double()
        x = s["logits"][b].double()
        x = torch.where(count > 0, x * s["repetition"][b].double() ** torch.where(x > 0, -1.0, 1.0), x)
        x = x - count * s["frequency"][b].double() - count.clamp(max=1) * s["presence"][b].double()
        allowed = (s["allowed"][b].long()[:, None] >> bits & 1).flatten()[: case["vocab"]]
        out[b] = (x + s["bias"][0].double()).masked_fill(allowed == 0, -math.inf)
    return [out, None]


def _books(s):
    return s["table"].tolist(), s["lengths"].tolist(), s["refcounts"].tolist()


def _as_tensors(table, lengths, refcounts):
    return [torch.tensor(table, dtype=torch.int32), torch.tensor(lengths), torch.tensor(refcounts, dtype=torch.int32)]


def _exact_admit(s, case):
    table, lengths, refcounts = _books(s)  # every slot is empty
    free = [p for p, held in enumerate(refcounts) if held == 0]
    for i, (slot, n) in enumerate(zip(s["slots"].tolist(), s["counts"].tolist())):
        for c in range(-(-n // case["page"])):
            p = free.pop(0)
            table[slot][c], refcounts[p] = p, 1
            rows = min(case["page"], n - c * case["page"])
            tokens = slice(c * case["page"], c * case["page"] + rows)
            s["key_pages"][p, :, :rows] = s["key"][i, :, tokens]
            s["value_pages"][p, :, :rows] = s["value"][i, :, tokens]
        lengths[slot] = n
    count = len(s["slots"])
    return [s["key_pages"], s["value_pages"], *_as_tensors(table, lengths, refcounts),
            torch.zeros(count, dtype=torch.int64), torch.zeros(count, dtype=torch.int32)]


def _exact_fork(s, case):
    table, lengths, refcounts = _books(s)  # every child is empty
    free = [p for p, held in enumerate(refcounts) if held == 0]
    for parent, child in zip(s["parents"].tolist(), s["children"].tolist()):
        full, rest = divmod(lengths[parent], case["page"])
        for c in range(full):
            table[child][c] = table[parent][c]
            refcounts[table[parent][c]] += 1
        if rest:
            p, last = free.pop(0), table[parent][full]
            table[child][full], refcounts[p] = p, 1
            s["key_pages"][:, p, :, :rest] = s["key_pages"][:, last, :, :rest]
            s["value_pages"][:, p, :, :rest] = s["value_pages"][:, last, :, :rest]
        lengths[child] = lengths[parent]
    return [s["key_pages"], s["value_pages"], *_as_tensors(table, lengths, refcounts),
            torch.zeros(len(s["parents"]), dtype=torch.int32)]


def _exact_compact(s, case):
    refcounts = s["refcounts"].tolist()
    used = sum(held > 0 for held in refcounts)
    page_map = [p if held else -1 for p, held in enumerate(refcounts)]
    holes = (p for p in range(used) if refcounts[p] == 0)
    for p in [p for p in range(used, len(refcounts)) if refcounts[p]]:
        to = next(holes)
        page_map[p] = to
        s["key_pages"][:, to] = s["key_pages"][:, p]
        s["value_pages"][:, to] = s["value_pages"][:, p]
    after = [0] * len(refcounts)
    for p, held in enumerate(refcounts):
        if held:
            after[page_map[p]] = held
    table = [[page_map[p] if p >= 0 else -1 for p in row] for row in s["table"].tolist()]
    return [s["key_pages"], s["value_pages"], torch.tensor(table, dtype=torch.int32),
            torch.tensor(after, dtype=torch.int32), torch.tensor(page_map, dtype=torch.int32), torch.tensor(used)]


def _exact_copy(s, case):
    for a, b in zip(s["source"].tolist(), s["target"].tolist()):
        s["key_pages"][:, b] = s["key_pages"][:, a]
        s["value_pages"][:, b] = s["value_pages"][:, a]
    return [s["key_pages"], s["value_pages"], torch.zeros(len(s["source"]), dtype=torch.int32)]


_EXACT = {"paged": _exact_paged, "window": _exact_window, "admit": _exact_admit, "fork": _exact_fork,
          "compact": _exact_compact, "copy": _exact_copy, "logits": _exact_logits}
