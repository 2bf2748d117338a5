"""Plain restatements of the serving operators: attention and logits in float64, pages as Python lists."""

from __future__ import annotations

import math

import torch


def visible_keys(position: int, length: int, window: int, sinks: int) -> list[int]:
    """Keys that the query at ``position`` of a sequence of ``length`` keys sees."""
    if not 0 <= position < length:
        return []
    return [j for j in range(position + 1) if window == 0 or j > position - window or j < sinks]


def attend(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, scale: float) -> torch.Tensor:
    """One row: query [D] over keys, values [n, D]."""
    if keys.shape[0] == 0:
        return torch.zeros(query.shape[0], dtype=torch.float64)
    scores = (keys.double() @ query.double()) * scale
    weights = torch.exp(scores - scores.max())
    return (weights @ values.double()) / weights.sum()


def paged_decode(query, key_pages, value_pages, page_table, lengths, scale, window=0, sinks=0, slots=None):
    batch, heads, _, dim = query.shape
    pages, kv_heads, page_size, _ = key_pages.shape
    out = torch.zeros(batch, heads, 1, dim, dtype=torch.float64)
    for b in range(batch):
        slot = b if slots is None else int(slots[b])
        if not 0 <= slot < page_table.shape[0]:
            continue
        n = max(0, min(int(lengths[slot]), page_table.shape[1] * page_size))
        rows = [(int(page_table[slot, j // page_size]), j % page_size) for j in visible_keys(n - 1, n, window, sinks)]
        rows = [(p, r) for p, r in rows if 0 <= p < pages]
        for h in range(heads):
            kv = h // (heads // kv_heads)
            p, r = [p for p, _ in rows], [r for _, r in rows]
            out[b, h, 0] = attend(query[b, h, 0], key_pages[p, kv, r], value_pages[p, kv, r], scale)
    return out


def window_attention(query, key, value, scale, window, sinks=0, lengths=None, starts=None):
    batch, heads, queries, dim = query.shape
    keys, group = key.shape[2], heads // key.shape[1]
    out = torch.zeros(batch, heads, queries, dim, dtype=torch.float64)
    for b in range(batch):
        n = keys if lengths is None else max(0, min(int(lengths[b]), keys))
        start = n - queries if starts is None else int(starts[b])
        for i in range(queries):
            seen = visible_keys(start + i, n, window, sinks)
            for h in range(heads):
                out[b, h, i] = attend(query[b, h, i], key[b, h // group, seen], value[b, h // group, seen], scale)
    return out


def attention_bound(query, keys, values, scale, terms: int, dtype: torch.dtype, expected: torch.Tensor,
                    rounded_weights: bool = False) -> torch.Tensor:
    """How far a result computed with float32 sums may be from ``expected``.

    A score is a sum of D products: it is off by at most (D + 2) 2^-24 times the sum of the magnitudes, itself at most
    |scale| |q| |k|; a matrix instruction may round a partial sum down instead of to nearest, which doubles the step.  A
    weight exp(s - m) is off, relative to itself, by the errors of s and m, by |s - m| 2^-23 for the scaled argument
    and by 2^-22 for the exponential, and a weight below 2^-40 does not count; a 16-bit weight kept in two terms by 2^-16
    more (bfloat16's two halves; a float16 weight loses 2^-22 of itself or, where it is small, 2^-37 of the largest weight,
    2^-36 where it has one term, which the step of the sums holds).  The two sums of ``terms`` weights are off by terms
    2^-23.  All of it moves a weighted mean of the values by at most twice the weights' relative error times the largest
    value.  The result is rounded once.

    ``rounded_weights``: 16-bit prompts round each weight p_j once to the type for its product with v_j, and sum the
    unrounded ones: sum p_j (1 + d_j) v_j / sum p_j with |d_j| at most half a step differs by at most half a step times
    the largest value.
    """
    dim = query.shape[-1]
    norms = query.double().norm(dim=-1).max() * keys.double().norm(dim=-1).max() * abs(scale)
    score = float((dim + 2) * 2.0 ** -23 * norms)
    weight = 2 * score + 40 * 2.0 ** -23 + 2.0 ** -22 + terms * 2.0 ** -23
    if dtype != torch.float32:
        weight += 2.0 ** -16
    largest = float(values.double().abs().max())
    half_step = torch.finfo(dtype).eps / 2
    smallest = torch.finfo(dtype).tiny
    if rounded_weights and dtype != torch.float32:
        weight += half_step / 2
    return 2 * weight * largest + half_step * expected.abs() + smallest


def processed_logits(logits, history=None, history_lengths=None, repetition=None, frequency=None, presence=None,
                     bias=None, allowed=None) -> torch.Tensor:
    """In float64, from the definition."""
    rows, vocab = logits.shape
    out = logits.double().clone()
    for b in range(rows):
        if history is not None:
            n = history.shape[1] if history_lengths is None else max(0, min(int(history_lengths[b]), history.shape[1]))
            count: dict[int, int] = {}
            for v in history[b, :n].tolist():
                if 0 <= v < vocab:
                    count[v] = count.get(v, 0) + 1
            for v, c in count.items():
                x = float(out[b, v])
                if repetition is not None:
                    x = x / float(repetition[b]) if x > 0 else x * float(repetition[b])
                if frequency is not None:
                    x -= float(frequency[b]) * c
                if presence is not None:
                    x -= float(presence[b])
                out[b, v] = x
        if bias is not None:
            out[b] += bias[b if bias.shape[0] > 1 else 0].double()
        if allowed is not None:
            words = allowed[b if allowed.shape[0] > 1 else 0].long()
            at = torch.arange(vocab)
            out[b][(words[at // 32] >> (at % 32)) & 1 == 0] = -math.inf
    return out


def greedy(processed: torch.Tensor) -> list[int]:
    """Lowest index of the largest value; NaN is above all numbers."""
    tokens = []
    for row in processed.double().tolist():
        nan = [i for i, x in enumerate(row) if x != x]
        tokens.append(nan[0] if nan else row.index(max(row)))
    return tokens


DONE, OUT_OF_RANGE, REPEATED, NO_ROOM, OCCUPIED = range(5)


class Pages:
    """The books and one row of K and V per position, as lists."""

    def __init__(self, layers, pages, heads, page_size, dim, slots, columns, dtype=torch.float32, seed=0):
        g = torch.Generator().manual_seed(seed)
        shape = (layers, pages, heads, page_size, dim)
        self.key, self.value = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
        self.table = [[-1] * columns for _ in range(slots)]
        self.lengths = [0] * slots
        self.refcounts = [0] * pages
        self.page_size = page_size
        self.pages, self.slots, self.columns = pages, slots, columns

    def _free_pages(self):
        return [p for p in range(self.pages) if self.refcounts[p] <= 0]

    def reserve(self, slots, counts):
        free, wanted = self._free_pages(), 0
        todo, positions, status = [], [], []
        for i, (slot, count) in enumerate(zip(slots, counts)):
            columns = []
            if not 0 <= slot < self.slots or count < 0:
                state = OUT_OF_RANGE
            elif slot in slots[:i]:
                state = REPEATED
            elif not 0 <= self.lengths[slot] <= self.columns * self.page_size:
                state = OUT_OF_RANGE
            elif count > self.columns * self.page_size - self.lengths[slot]:
                state = NO_ROOM
            else:
                state = DONE
                used = {p // self.page_size for p in range(self.lengths[slot], self.lengths[slot] + count)}
                columns = [c for c in sorted(used) if self.table[slot][c] < 0]
                wanted += len(columns)
                if columns and wanted > len(free):
                    state = NO_ROOM
            positions.append(self.lengths[slot] if state == DONE else -1)
            status.append(state)
            if state == DONE:
                todo.append((slot, count, columns))
        for slot, count, columns in todo:
            for c in columns:
                self.table[slot][c] = free.pop(0)
                self.refcounts[self.table[slot][c]] = 1
            self.lengths[slot] += count
        return positions, status

    def write(self, layer, key, value, slots, positions, counts):
        for i, (slot, start) in enumerate(zip(slots, positions)):
            if not 0 <= slot < self.slots or start < 0:
                continue
            for t in range(min(key.shape[2], counts[i])):
                column = (start + t) // self.page_size
                page = self.table[slot][column] if column < self.columns else -1
                if 0 <= page < self.pages:
                    self.key[layer, page, :, (start + t) % self.page_size] = key[i, :, t]
                    self.value[layer, page, :, (start + t) % self.page_size] = value[i, :, t]

    def copy(self, source, target):
        status = []
        for i, (a, b) in enumerate(zip(source, target)):
            if not (0 <= a < self.pages and 0 <= b < self.pages):
                status.append(OUT_OF_RANGE)
            elif b in target[:i] or any(s == b for j, s in enumerate(source) if j != i):
                status.append(REPEATED)
            else:
                status.append(DONE)
        for a, b, state in zip(source, target, status):
            if state == DONE:
                self.key[:, b], self.value[:, b] = self.key[:, a].clone(), self.value[:, a].clone()
        return status

    def free(self, slots):
        status = []
        for i, slot in enumerate(slots):
            if not 0 <= slot < self.slots:
                status.append(OUT_OF_RANGE)
            elif slot in slots[:i]:
                status.append(REPEATED)
            else:
                status.append(DONE)
                for p in self.table[slot]:
                    if 0 <= p < self.pages:
                        self.refcounts[p] = max(0, self.refcounts[p] - 1)
                self.table[slot] = [-1] * self.columns
                self.lengths[slot] = 0
        return status

    def fork(self, parents, children):
        free, wanted = self._free_pages(), 0
        before = [list(row) for row in self.table], list(self.lengths)
        status = []
        for i, (parent, child) in enumerate(zip(parents, children)):
            state = DONE
            if not (0 <= parent < self.slots and 0 <= child < self.slots):
                state = OUT_OF_RANGE
            elif child in [c for c in children[:i]]:
                state = REPEATED
            elif before[1][child] != 0 or any(p >= 0 for p in before[0][child]):
                state = OCCUPIED
            elif not 0 <= before[1][parent] <= self.columns * self.page_size or any(
                    not 0 <= p < self.pages for p in before[0][parent][: -(-before[1][parent] // self.page_size)]):
                state = OUT_OF_RANGE
            if state == DONE:
                full, rest = divmod(before[1][parent], self.page_size)
                wanted += rest > 0
                if rest and wanted > len(free):
                    state = NO_ROOM
            status.append(state)
            if state != DONE:
                continue
            for c in range(full):
                self.table[child][c] = before[0][parent][c]
                self.refcounts[before[0][parent][c]] += 1
            if rest:
                page, last = free[wanted - 1], before[0][parent][full]
                self.table[child][full] = page
                self.refcounts[page] = 1
                self.key[:, page, :, :rest] = self.key[:, last, :, :rest]
                self.value[:, page, :, :rest] = self.value[:, last, :, :rest]
            self.lengths[child] = before[1][parent]
        return status

    def compact(self):
        used = sum(c > 0 for c in self.refcounts)
        holes = [p for p in range(used) if self.refcounts[p] <= 0]
        movers = [p for p in range(used, self.pages) if self.refcounts[p] > 0]
        page_map = [p if c > 0 else -1 for p, c in enumerate(self.refcounts)]
        for a, b in zip(movers, holes):
            page_map[a] = b
            self.key[:, b], self.value[:, b] = self.key[:, a].clone(), self.value[:, a].clone()
            self.refcounts[b], self.refcounts[a] = self.refcounts[a], 0
        self.table = [[(page_map[p] if p < self.pages else -1) if p >= 0 else p for p in row] for row in self.table]
        return page_map, used
