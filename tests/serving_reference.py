"""Plain forms of the operators around a decoding step with drafts, for their tests:
verification of drafts and low-rank adapters in float64 on the CPU, the pool's book in
Python lists.  Written from the definitions."""

from __future__ import annotations

import math

import torch

BLOCK = 64


def probabilities(logits, temperature):
    """softmax(logits / temperature) of one row in float64 (temperature None, or not
    above 0: all at the first of the largest), or None for a row without any."""

    logits = logits.double()
    if bool(torch.isnan(logits).any()) or not math.isfinite(float(logits.max())):
        return None
    if not temperature > 0:
        first = int((logits == logits.max()).nonzero()[0, 0])
        return torch.zeros_like(logits).index_fill_(0, torch.tensor([first]), 1.0)
    away = logits - logits.max()
    # an infinite temperature: alike for all that is not masked
    weights = torch.exp(torch.where(torch.isinf(away), away, away / temperature))
    return weights / weights.sum()


def verify(target, tokens, uniforms, draft, counts, temperatures):
    """CPU tensors of the operator's arguments; answer, accepted as lists."""

    batch, drafts = tokens.shape
    answers, accepted = [], []
    for b in range(batch):
        count = drafts if counts is None else min(int(counts[b]), drafts)
        temperature = 1.0 if temperatures is None else float(temperatures[b])
        if count < 0:
            answers.append([-1] * (drafts + 1))
            accepted.append(-1)
            continue
        kept, weights = 0, None
        while True:
            p = probabilities(target[b, kept], temperature)
            if kept == count or p is None:
                weights = p
                break
            x = int(tokens[b, kept])
            known = 0 <= x < p.numel()
            q = torch.zeros_like(p)
            if draft is not None and temperature > 0:
                q = probabilities(draft[b, kept], temperature)
            elif known:
                q[x] = 1.0
            if q is None:
                break
            if known and float(uniforms[b, kept]) * float(q[x]) < float(p[x]):
                kept += 1
                continue
            weights = (p - q).clamp(min=0)
            break
        chosen = -1
        if weights is not None and float(weights.sum()) > 0:
            sums = weights.cumsum(0)
            above = ((sums > float(uniforms[b, drafts]) * float(sums[-1])) & (weights > 0)).nonzero()
            chosen = int(above[0, 0]) if above.numel() else int((weights > 0).nonzero()[-1, 0])
        answers.append(tokens[b, :kept].tolist() + [chosen] + [-1] * (drafts - kept))
        accepted.append(kept)
    return answers, accepted


def adapters(value, projected, down, up, scales, ranks, indices, counts):
    """[batch, seq, features] in any type; the sum in float64, and the magnitudes of
    its two inner sums: of the products x down (through up), and of h alone."""

    out = projected.double()
    terms, hidden_size = torch.zeros_like(out), torch.zeros_like(out)
    for b, index in enumerate(indices.tolist()):
        if not 0 <= index < down.shape[0]:
            continue
        count = out.shape[1] if counts is None else max(0, min(int(counts[b]), out.shape[1]))
        rank = down.shape[1] if ranks is None else max(0, min(int(ranks[index]), down.shape[1]))
        if rank == 0 or count == 0:
            continue
        scale = 1.0 if scales is None else float(scales[index])
        x = value[b, :count].double()
        d, u = down[index, :rank].double(), up[index, :, :rank].double()
        hidden = x @ d.t()
        out[b, :count] += scale * (hidden @ u.t())
        terms[b, :count] = abs(scale) * ((x.abs() @ d.abs().t()) @ u.abs().t())
        hidden_size[b, :count] = abs(scale) * hidden.abs().amax(-1, keepdim=True) * u.abs().sum(-1)
    return out, terms, hidden_size


def adapters_bound(out, terms, hidden_size, in_features, rank, dtype):
    """The output's rounding; fp32 sums of ``in_features`` and of ``rank`` products
    (twice, high and low part); and h as two numbers of dtype: each is rounded by half a
    step of its own, together half a step squared of h (in fp16 no finer than 2^-25 of a
    unit in which the token's largest h is 2^14 or more, 2^-39 of it).  The magnitudes
    may come out a little below a rounded h's own: a factor of 1.01."""

    step = torch.finfo(dtype).eps / 2
    inner = (in_features + 2 * rank + 16) * 2.0**-24 * terms + (step * step + 2.0**-38) * hidden_size
    inner = 1.01 * inner
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2  # half a subnormal step
    return step * (out.abs() + inner) + inner + least


class Book:
    """The pool as lists: the table's rows and the holders."""

    def __init__(self, table, holders):
        self.table, self.holders = [list(row) for row in table], list(holders)

    def is_place(self, place):
        return 0 <= place < len(self.holders)

    def reserve(self, starts, tokens, counts=None):
        missing = []
        for b, start in enumerate(starts):
            count = tokens if counts is None else min(counts[b], tokens)
            lacking = 0
            if start >= 0 and count > 0:
                for block in range(start // BLOCK, (start + count) // BLOCK):
                    if block >= len(self.table[b]):
                        lacking += 1
                        continue
                    if self.is_place(self.table[b][block]):
                        continue
                    free = [p for p, held in enumerate(self.holders) if held <= 0]
                    if not free:
                        lacking += 1
                        continue
                    self.table[b][block] = free[0]
                    self.holders[free[0]] = 1
            missing.append(lacking)
        return missing

    def release(self, lengths):
        for b, length in enumerate(lengths):
            if length < 0:
                continue
            for block in range(length // BLOCK, len(self.table[b])):
                if self.is_place(self.table[b][block]):
                    self.holders[self.table[b][block]] -= 1
                self.table[b][block] = -1

    def fork(self, sources, lengths):
        before = [list(row) for row in self.table]
        for b, source in enumerate(sources):
            if not 0 <= source < len(before) or source == b:
                continue
            whole = max(lengths[source], 0) // BLOCK
            self.table[b] = [p if block < whole else -1 for block, p in enumerate(before[source])]
            for p in before[b]:
                if self.is_place(p):
                    self.holders[p] -= 1
            for p in self.table[b]:
                if self.is_place(p):
                    self.holders[p] += 1

    def compact(self):
        used = [p for p, held in enumerate(self.holders) if held > 0]
        holes = [p for p in range(len(used)) if self.holders[p] <= 0]
        moves = dict(zip([p for p in used if p >= len(used)], holes))
        origins = [-1] * len(self.holders)
        for mover, hole in moves.items():
            origins[hole] = mover
            self.holders[hole], self.holders[mover] = self.holders[mover], 0
        self.table = [[moves.get(p, p) for p in row] for row in self.table]
        return origins, len(used)


class TokenCache:
    """Token numbers where a layer's cache holds keys and values: a tail of 64 a sequence, the
    places' blocks, and the book's table.  LOST is what nobody can read back."""

    LOST = -1

    def __init__(self, book):
        self.book = book
        self.tails = [[self.LOST] * BLOCK for _ in book.table]
        self.places = [[self.LOST] * BLOCK for _ in book.holders]

    def _place(self, b, block):
        row = self.book.table[b]
        place = row[block] if block < len(row) else -1
        return place if self.book.is_place(place) else None

    def append(self, starts, counts, tokens):
        for b, (start, count) in enumerate(zip(starts, counts)):
            for i in range(count):
                self.tails[b][(start + i) % BLOCK] = tokens[b][i]
                place = self._place(b, (start + i) // BLOCK)
                if (start + i) % BLOCK == BLOCK - 1 and place is not None:
                    self.places[place] = list(self.tails[b])

    def read(self, b, length):
        held = []
        for block in range(length // BLOCK):
            place = self._place(b, block)
            held += [self.LOST] * BLOCK if place is None else self.places[place]
        return held + self.tails[b][: length % BLOCK]

    def take_back(self, lengths, ends):
        for b, (length, end) in enumerate(zip(lengths, ends)):
            if end >= 0 and end % BLOCK and end // BLOCK < length // BLOCK:
                place = self._place(b, end // BLOCK)
                self.tails[b] = [self.LOST] * BLOCK if place is None else list(self.places[place])

    def fork(self, sources):
        before = self.tails
        self.tails = [list(before[s if 0 <= s < len(before) else b]) for b, s in enumerate(sources)]

    def copy(self, origins):
        before = [list(place) for place in self.places]
        for target, origin in enumerate(origins):
            if origin >= 0:
                self.places[target] = before[origin]
