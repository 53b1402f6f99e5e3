"""Paged caches and token sampling in plain numpy and Python, for the tests."""

from __future__ import annotations

import math

import numpy as np
import torch

from .cache4_reference import attend

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# 16-bit weights are kept as two terms, the second the rounded rest of the first: each within half a step of half a step
# (an fp16 weight under the normal range, 2^-14 of a reference kept at 2^8, within 2^-25 of 2^8 too)
WEIGHTS = {torch.float32: 2.0 ** -22, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22}


def check_attention(got, q, keys, values, allowed, scaling):
    """got / q [R, D] of one head over keys / values [N, D] (tensors), allowed [R, N]: within the errors of fp32 scores
    and sums (cache4_reference.attend), the weights' two terms and the output's rounding."""
    K, V, x = (t.double().cpu().numpy() for t in (keys, values, q))
    ref, bound = attend(x, K, V, allowed, scaling)
    size, _ = attend(x, K, np.abs(V), allowed, scaling)
    extra = WEIGHTS[q.dtype] * size
    if q.dtype == torch.float16 and len(K):
        extra = extra + 2.0 ** -33 * len(K) * np.abs(V).max()
    over = np.abs(got.double().cpu().numpy() - ref) - bound - extra - HALF_STEP[got.dtype] * np.abs(ref)
    assert (over <= 1e-30).all(), f"over the bound by {np.nanmax(over)}"


class Holder:
    """Page tables in Python: what pages_reserve, pages_fork and pages_compact do, and every sequence's rows by value."""

    def __init__(self, n_seq, entries, pages, page_rows):
        self.held, self.lens, self.rows = [[] for _ in range(n_seq)], [0] * n_seq, [[] for _ in range(n_seq)]
        self.entries, self.pages, self.P = entries, pages, page_rows

    def refs(self):
        count = [0] * self.pages
        for h in self.held:
            for p in h:
                count[p] += 1
        return count

    def reserve(self, counts):
        """(first rows, pairs); `rows` is left to the caller's writes."""
        refs = self.refs()
        free = [p for p, r in enumerate(refs) if r == 0]
        room, asked, first, pairs, new = len(free), 0, [], [], []
        for held, n, c in zip(self.held, self.lens, counts):
            pair, want = (-1, -1), None
            if c >= 0 and n + c <= self.entries * self.P:
                parts = c > 0 and n % self.P != 0 and refs[held[-1]] > 1
                need = math.ceil((n + c) / self.P) - len(held) + parts
                asked += need
                if need == 0 or asked <= room:
                    got = free[asked - need:asked]
                    if parts:
                        pair, held = (held[-1], got[0]), held[:-1]
                    want = held + got
            first.append(-1 if want is None else n)
            pairs.append(pair)
            new.append(want)
        for i, want in enumerate(new):
            if want is not None:
                self.held[i], self.lens[i] = want, self.lens[i] + counts[i]
        return first, pairs

    def fork(self, sources):
        old = [(list(h), n, list(r)) for h, n, r in zip(self.held, self.lens, self.rows)]
        for i, s in enumerate(sources):
            if s == -1:
                self.held[i], self.lens[i], self.rows[i] = [], 0, []
            elif 0 <= s < len(old) and s != i:
                self.held[i], self.lens[i], self.rows[i] = list(old[s][0]), old[s][1], list(old[s][2])

    def compact(self):
        refs = self.refs()
        used = sum(r > 0 for r in refs)
        pairs = list(zip([p for p in range(used, self.pages) if refs[p]], [p for p in range(used) if not refs[p]]))
        to = dict(pairs)
        self.held = [[to.get(p, p) for p in h] for h in self.held]
        return pairs, used


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, border=0.0):
    """The next token of one row of float64 logits; None where the answer lies within `border` (of the sum) of another's
    share, a cut by top_p included."""
    x = np.where(np.isnan(logits), -np.inf, logits)
    top = x.max()
    if top == -np.inf:
        return -1
    if temperature <= 0 or top_k == 1:
        return int(np.argmax(x))
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / temperature))
    order = np.lexsort((np.arange(len(x)), -x))  # falling, ties by number
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        share = np.cumsum(w[order])
        before, total = share - w[order], share[-1]
        if border and np.min(np.abs(before[1:] - top_p * total), initial=np.inf) < border * total:
            return None
        keep = before < top_p * total
        keep[0] = True
        order = order[keep]
    kept = np.zeros(len(x))
    order = order[w[order] >= min_p]
    kept[order] = w[order]
    share = np.cumsum(kept)
    at = u * share[-1]
    i = min(int(np.searchsorted(share, at, side="right")), int(np.flatnonzero(kept)[-1]))
    if border and np.min(np.abs(share - at)) < border * share[-1] and at > 0:
        return None
    return i
