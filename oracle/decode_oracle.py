"""CPU restatement of what a decoding loop does around the key/value cache: pages
handed out and shared, rotary positions, beam search's selection.  Written from the
definitions, one sequence, row or candidate at a time."""
from __future__ import annotations

import math
from fractions import Fraction

import numpy as np
import torch

PI = Fraction(3141592653589793238462643383279502884197169399375105820974944592, 10 ** 63)


class PageBook:
    """A pool's state and calls.  ``pages[s]``: the pages of sequence s."""

    def __init__(self, blocks: int, page: int, seqs: int, width: int):
        self.blocks, self.page, self.seqs, self.width = blocks, page, seqs, width
        self.refs = [0] * blocks
        self.pages = [[] for _ in range(seqs)]
        self.lengths = [0] * seqs

    def _for(self, tokens: int) -> int:
        return -(-tokens // self.page)

    def table(self) -> torch.Tensor:
        return torch.tensor([p + [-1] * (self.width - len(p)) for p in self.pages], dtype=torch.int32)

    def trim(self, to) -> None:
        for s, n in enumerate(to):
            self.lengths[s] = min(self.lengths[s], max(int(n), 0))
            while len(self.pages[s]) > self._for(self.lengths[s]):
                self.refs[self.pages[s].pop()] -= 1

    def reorder(self, parents) -> None:
        new = [list(self.pages[p]) if 0 <= p < self.seqs else [] for p in parents]
        lengths = [self.lengths[p] if 0 <= p < self.seqs else 0 for p in parents]
        for held, change in ((new, 1), (self.pages, -1)):
            for pages in held:
                for p in pages:
                    self.refs[p] += change
        self.pages, self.lengths = new, lengths

    def assign(self, new, rows: int, max_query: int, max_length: int):
        """lengths, starts, copies and missing of the step."""
        new = [min(max(int(n), 0), max_query) for n in new]
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        nothing = ([0] * self.seqs, starts, [(-1, -1, 0)] * self.seqs)
        room = min(self.width * self.page, max_length)
        if starts[-1] > rows:
            return (*nothing, -2)
        if any(n > room - old for n, old in zip(new, self.lengths) if n):
            return (*nothing, -1)
        going = {}
        for s, n in enumerate(new):
            if n and self.lengths[s] % self.page:
                going.setdefault(self.pages[s][-1], []).append(s)
        copied = [bool(n and self.lengths[s] % self.page and self.refs[self.pages[s][-1]] > 1
                       and not (len(going[self.pages[s][-1]]) == self.refs[self.pages[s][-1]] and going[self.pages[s][-1]][0] == s))
                  for s, n in enumerate(new)]
        wanted = sum(self._for(old + n) - self._for(old) + c for old, n, c in zip(self.lengths, new, copied) if n)
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if wanted > len(free):
            return (*nothing, wanted - len(free))
        free = iter(free)
        copies = []
        for s, n in enumerate(new):
            copies.append((-1, -1, 0))
            if copied[s]:
                old, page = self.pages[s][-1], next(free)
                copies[s] = (old, page, self.lengths[s] % self.page)
                self.pages[s][-1] = page
                self.refs[page] += 1
                self.refs[old] -= 1
            if n:
                self.lengths[s] += n
                while len(self.pages[s]) < self._for(self.lengths[s]):
                    self.pages[s].append(next(free))
                    self.refs[self.pages[s][-1]] += 1
        return [old if n else 0 for old, n in zip(self.lengths, new)], starts, copies, 0


def slots(table, lengths, starts, rows: int, page: int, blocks: int, max_query: int, max_length: int):
    """Positions and slots of a batch's rows; ``starts`` None: a row each."""
    positions, places = [0] * rows, [-1] * rows
    for s, n in enumerate(lengths):
        first = s if starts is None else min(max(int(starts[s]), 0), rows)
        last = s + 1 if starts is None else min(max(int(starts[s + 1]), first), rows)
        for row in range(first, last):
            at = max(int(n), 0) - (last - first) + (row - first)
            positions[row] = max(at, 0)
            if at < 0 or row - first >= max_query or at >= max_length:
                continue
            number = int(table[s][at // page])
            if 0 <= number < blocks:
                places[row] = number * page + at % page
    return torch.tensor(positions, dtype=torch.int32), torch.tensor(places, dtype=torch.int64)


def rotary_angles(frequencies, positions) -> tuple[torch.Tensor, torch.Tensor]:
    """Cosines and sines in 64 bits, the fraction of a turn from whole numbers."""
    turns = [[float(Fraction(f) * int(p) / (2 * PI) % 1) for f in frequencies] for p in positions]
    angle = torch.tensor(turns, dtype=torch.float64).view(len(turns), 1, -1) * (2 * math.pi)
    return angle.cos(), angle.sin()


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool, magnitude: float = 1.0) -> torch.Tensor:
    """x [rows, heads, dim] in 64 bits; the gradient takes -sin."""
    n = cos.shape[-1]
    y = x.double().clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    u, v = x.double()[..., first], x.double()[..., second]
    y[..., first] = magnitude * (u * cos - v * sin)
    y[..., second] = magnitude * (v * cos + u * sin)
    return y


def beam_scores(logits: torch.Tensor, scores: torch.Tensor, finished, end_token) -> torch.Tensor:
    """Scores of all continuations [requests, beams, vocabulary] in 64 bits, minus infinity: no candidate."""
    x = logits.double()
    out = torch.full(x.shape, -math.inf, dtype=torch.float64)
    for r in range(x.shape[0]):
        for b in range(x.shape[1]):
            own = float(scores[r, b])
            if finished is not None and bool(finished[r, b]):
                if math.isfinite(own):
                    out[r, b, end_token] = own
                continue
            row = x[r, b]
            if not math.isfinite(own) or bool(torch.isnan(row).any()) or not math.isfinite(float(row.max())):
                continue
            out[r, b] = own + (row - torch.logsumexp(row, 0))
    return out


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int, finished=None, end_token=None):
    """Scores in 64 bits, tokens and parents [requests, k]."""
    requests, beams, size = logits.shape
    all_scores = beam_scores(logits, scores, finished, end_token).numpy()
    out = []
    for r in range(requests):
        found = []
        for b in range(beams):
            row = all_scores[r, b]
            order = logits[r, b].double().numpy()
            if finished is not None and bool(finished[r, b]):
                order = row
            keep = np.nonzero(np.isfinite(row))[0]
            best = keep[np.lexsort((keep, -order[keep]))][:k]  # the larger logit, then the lower token
            found += [(-row[v], b, i, int(v)) for i, v in enumerate(best)]
        found.sort()
        found = [(-s, v, r * beams + b) for s, b, _, v in found[:k]]
        found += [(-math.inf, 0 if end_token is None else end_token, r * beams + j % beams) for j in range(len(found), k)]
        out.append(found)
    pick = [[[c[i] for c in found] for found in out] for i in range(3)]
    return (torch.tensor(pick[0], dtype=torch.float64).view(requests, k), torch.tensor(pick[1], dtype=torch.int32).view(requests, k),
            torch.tensor(pick[2], dtype=torch.int32).view(requests, k))
