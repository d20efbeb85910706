"""64-bit NumPy definitions of the verify step's operators, for tests: query/key preparation, tree attention over a
paged cache, acceptance of drafted tokens and the commit of the accepted ones."""
from __future__ import annotations

import numpy as np


def rope_table(positions, rotary, base):
    angle = np.arange(positions, dtype=np.float64)[:, None] * base ** (-2.0 * np.arange(rotary // 2) / rotary)
    return np.stack([np.cos(angle), np.sin(angle)], axis=2)


def norm_rope(x, weight, eps, table_rows, rotary):
    """x [rows][heads][d] -> normalised and rotated; table_rows [rows][rotary/2][2]."""
    x = np.asarray(x, np.float64)
    y = x / np.sqrt((x * x).mean(axis=2, keepdims=True) + eps) * np.asarray(weight, np.float64)
    if rotary:
        half = rotary // 2
        cos, sin = (np.asarray(table_rows, np.float64)[:, None, :, i] for i in (0, 1))
        a, b = y[..., :half].copy(), y[..., half:rotary].copy()
        y[..., :half], y[..., half:rotary] = a * cos - b * sin, b * cos + a * sin
    return y


def positions_rows(table, page, start, count):
    """Pool rows of `count` positions from `start` on, of the sequence whose page-table row is `table`."""
    p = np.arange(start, start + count)
    return np.asarray(table)[p // page] * page + p % page


def attention(q, k_rows, v_rows, masks, scale):
    """One sequence: q [tokens][hq][d]; k_rows, v_rows [length + tokens][hkv][d]; masks: one integer of node bits per
    token. What a token does not see is left out of its sums altogether."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k_rows, v_rows))
    tokens, hq, d = q.shape
    length, hkv = k.shape[0] - tokens, k.shape[1]
    out = np.zeros((tokens, hq, d))
    for t in range(tokens):
        seen = np.concatenate([np.arange(length), [length + j for j in range(tokens) if int(masks[t]) >> j & 1]]).astype(int)
        if not len(seen):
            continue
        for h in range(hq):
            g = h // (hq // hkv)
            with np.errstate(all="ignore"):
                s = k[seen, g] @ q[t, h] * scale
                w = np.exp(s - s.max())
                out[t, h] = w @ v[seen, g] / w.sum()
    return out


def chain_masks(tokens):
    return [(2 << i) - 1 for i in range(tokens)]


def tree_masks(parents):
    masks = []
    for i, p in enumerate(parents):
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
    return masks


def target(row, temperature):
    row = np.asarray(row, np.float64)
    if temperature == 0:
        p = np.zeros_like(row)
        p[int(row.argmax())] = 1.0
        return p
    w = np.exp((row - row.max()) / temperature)
    return w / w.sum()


def verify(logits, draft, parents, probs, uniforms, temperature):
    """One sequence. Returns (path, next token, margin): margin is how far the nearest decision was from its limit,
    relative to the mass it was made on."""
    tokens = len(parents)
    uniforms = np.asarray(uniforms, np.float64)
    path, at, margin = [0], 0, 1.0
    while True:
        p, chosen = target(logits[at], temperature), None
        for c in (c for c in range(1, tokens) if parents[c] == at):
            if probs is None:
                limit, mass = p[draft[c]], p.sum()
            else:
                limit, mass = p[draft[c]], float(probs[c][draft[c]])
            if mass > 0:
                margin = min(margin, abs(uniforms[c] * mass - limit) / mass)
            if uniforms[c] * mass < limit:
                chosen = c
                break
            if probs is None:
                p[draft[c]] = 0.0
            else:
                left = np.maximum(p - np.asarray(probs[c], np.float64), 0.0)
                p = left / left.sum() if left.sum() > 0 else p
        if chosen is None:
            break
        at = chosen
        path.append(at)
    run = np.cumsum(p)
    aim = uniforms[0] * run[-1]
    pick = int((run <= aim).sum())
    steps = run[p > 0]  # where the pick changes
    margin = min(margin, float(np.abs(np.concatenate([[0.0] if aim > 0 else [], steps[:-1]]) - aim).min() / run[-1]) if len(steps) > 1 else margin)
    return path, pick, margin
