"""64-bit NumPy definitions of the operators for a batch of users, for tests: what sampling settings keep of a row of logits,
the next token, and the hand-out of a paged cache's pages."""
from __future__ import annotations

import numpy as np


def kept(row, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Indices that may be drawn, best first, their weights relative to the largest, and how far the nearest border of a sum
    was from it, relative to the sum. None for a row that is refused."""
    row = np.asarray(row, np.float64)
    if np.isnan(row).any() or (row == np.inf).any() or not np.isfinite(row).any():
        return None
    if not 0 <= temperature < np.inf or np.isnan(top_p) or np.isnan(min_p):
        return None
    best = np.flatnonzero(row > -np.inf)
    best = best[np.argsort(-row[best], kind="stable")]
    if temperature == 0:
        return best[:1], np.ones(1), 1.0
    with np.errstate(under="ignore"):
        w = np.exp((row[best] - row[best[0]]) / float(temperature))
    margin = 1.0
    if top_k > 0:
        best, w = best[:top_k], w[:top_k]
    if top_p < 1:
        upto = np.cumsum(w)
        n = max(1, int((upto - w < top_p * upto[-1]).sum()))
        margin = float(np.abs(upto - top_p * upto[-1]).min() / upto[-1])
        best, w = best[:n], w[:n]
    n = max(1, int((w >= min_p).sum()))
    return best[:n], w[:n], margin


def sample(row, uniform, **settings):
    """(token, margin); -1 for a row that is refused."""
    found = None if np.isnan(uniform) else kept(row, **settings)
    if found is None:
        return -1, 1.0
    best, w, margin = found
    order = np.argsort(best)
    upto = np.cumsum(w[order])
    aim = min(max(float(uniform), 0.0), 1 - 2.0 ** -24) * upto[-1]
    token = int(best[order][min(len(order) - 1, int((upto <= aim).sum()))])
    if len(order) > 1:
        margin = min(margin, float(np.abs(upto[:-1] - aim).min() / upto[-1]))
    return token, margin


class Pages:
    """The page tables and the stack of free pages, on the host."""

    def __init__(self, table, held, stack, page):
        self.table, self.held, self.stack, self.page = [list(map(int, r)) for r in table], list(map(int, held)), list(map(int, stack)), page

    def reserve(self, lengths, counts, tokens, pages):
        taken, slots, short = [], [], False
        for s, (n, c) in enumerate(zip(lengths, counts)):
            none = [-1] * tokens
            room = len(self.table[s])
            if n < 0 or not 0 <= c <= tokens or n + c > room * self.page or not 0 <= self.held[s] <= room:
                taken.append(-1)
                slots.append(none)
                continue
            need = max(0, -(-(n + c) // self.page) - self.held[s])
            short = short or need > len(self.stack)
            if short and need:
                taken.append(-2)
                slots.append(none)
                continue
            for _ in range(need):
                self.table[s][self.held[s]] = self.stack.pop()
                self.held[s] += 1
            taken.append(need)
            at = [(self.table[s][p // self.page], p % self.page) for p in range(n, n + c)]
            slots.append([q * self.page + r if 0 <= q < pages else -1 for q, r in at] + none[c:])
        return taken, slots

    def release(self, lengths, shared_pages, pages):
        back, freed, held = [], [], []
        for s, n in enumerate(lengths):
            h = self.held[s]
            if not 0 <= h <= len(self.table[s]):
                freed.append(-1)
                held.append(h)
                continue
            stay = min(h, max(shared_pages, -(-max(n, 0) // self.page)))
            back += self.table[s][stay:h]
            freed.append(h - stay)
            held.append(stay)
        if len(self.stack) + len(back) > pages:
            return [-1 if f else 0 for f in freed]
        self.stack += back[::-1]
        self.held = held
        return freed
