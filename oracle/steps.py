"""Plain restatements of the operators of mixed steps: lists for what counts, float64 for attention, fractions for sampling."""

from __future__ import annotations

import math
from fractions import Fraction

import torch


def step_layout(page_table, slots, positions, counts, page_size, tokens):
    """(offsets, requests, positions, rows) as lists."""
    table = page_table.tolist()
    offsets, request, position, row = [0], [], [], []
    for i, (slot, first) in enumerate(zip(slots.tolist(), positions.tolist())):
        count = 1 if counts is None else int(counts[i])
        if first < 0 or not 0 <= slot < len(table) or count < 0:
            count = 0
        for p in range(first, first + min(count, tokens - len(request))):
            page = table[slot][p // page_size] if p // page_size < len(table[0]) else -1
            request.append(i)
            position.append(p)
            row.append(page * page_size + p % page_size if page >= 0 else -1)
        offsets.append(len(request))
    behind = [-1] * (tokens - len(request))
    return offsets, request + behind, position + behind, row + behind


def write_rows(key, value, key_pages, value_pages, rows):
    """In place."""
    pages, _, page_size, _ = key_pages.shape
    for t, r in enumerate(rows.tolist()):
        if 0 <= r < pages * page_size:
            key_pages[r // page_size, :, r % page_size] = key[t]
            value_pages[r // page_size, :, r % page_size] = value[t]


def chunk_attention(query, key_pages, value_pages, page_table, lengths, offsets, scale, window=0, sinks=0, slots=None,
                    positions=None):
    tokens, heads, dim = query.shape
    pages, kv_heads, page_size, _ = key_pages.shape
    group = heads // kv_heads
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64)
    for i in range(len(offsets) - 1):
        low, high = int(offsets[i]), int(offsets[i + 1])
        slot = i if slots is None else int(slots[i])
        begin, end = max(0, min(low, tokens)), max(0, min(high, tokens))
        if not 0 <= slot < page_table.shape[0] or begin >= end:
            continue
        n = max(0, min(int(lengths[slot]), page_table.shape[1] * page_size))
        first = n - (high - low) if positions is None else int(positions[i])
        p = first + torch.arange(end - begin)[:, None]
        j = torch.arange(n)
        page = page_table[slot, j // page_size].long()
        seen = (j <= p) & (p >= 0) & (p < n) & (page >= 0) & (page < pages)
        if window:
            seen &= (j > p - window) | (j < sinks)
        some = seen.any(0).nonzero()[:, 0]
        if len(some) == 0:
            continue
        seen = seen[:, some]
        for h in range(heads):
            key = key_pages[page[some], h // group, some % page_size].double()
            value = value_pages[page[some], h // group, some % page_size].double()
            for r in range(end - begin):  # a row reads the keys that it sees, and no others
                mine = seen[r]
                if not mine.any():
                    continue
                score = (key[mine] @ query[begin + r, h].double()) * scale
                if score.max() == -math.inf:
                    continue
                weight = torch.exp(score - score.max())
                out[begin + r, h] = (weight @ value[mine]) / weight.sum()
    return out


def sample(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None):
    """(tokens, probabilities) by exact sums of the float64 weights."""
    tokens, probabilities = [], []
    for b, row in enumerate(logits.double().tolist()):
        t = 1.0 if temperature is None else float(temperature[b])
        nan = [i for i, x in enumerate(row) if x != x]
        best = nan[0] if nan else row.index(max(row))
        if not t > 0 or not math.isfinite(row[best]):
            tokens.append(best)
            probabilities.append(1.0)
            continue
        weight = [0.0 if x == -math.inf else math.exp((x - row[best]) / t) for x in row]
        kept = sorted(range(len(row)), key=lambda v: (-row[v], v))
        if top_k is not None and int(top_k[b]) > 0:
            kept = kept[: int(top_k[b])]
        if top_p is not None and float(top_p[b]) < 1:
            limit = Fraction(max(float(top_p[b]), 0.0)) * sum(Fraction(weight[v]) for v in kept)
            before, count = Fraction(0), 0
            for v in kept:
                if count and before >= limit:
                    break
                before += Fraction(weight[v])
                count += 1
            kept = kept[:count]
        if min_p is not None and float(min_p[b]) > 0:
            kept = [v for v in kept if weight[v] >= min(float(min_p[b]), 1.0)]
        all_of_them = sum(Fraction(weight[v]) for v in kept)
        u = float(uniforms[b])
        target = Fraction(u) * all_of_them if u > 0 else Fraction(0)
        reached, token = Fraction(0), None
        for v in sorted(kept):
            if weight[v] == 0:
                continue
            reached += Fraction(weight[v])
            token = v
            if reached > target:
                break
        tokens.append(token)
        probabilities.append(float(Fraction(weight[token]) / all_of_them))
    return tokens, probabilities
