"""The paged 4-bit cache in numpy, 64 bits: the values, the tables and the attention, each from its definition
(include/dimmerkv.h) and one step at a time.  No counterpart in the reference."""

from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
EXP_MIN, EXP_MAX, NAN = -22, 13, 255


def quantize(rows: np.ndarray):
    """[..., D] -> codes uint8 [..., D], scale bytes uint8 [..., D / 32], values float64 [..., D]."""
    rows = np.asarray(rows, dtype=np.float64)
    blocks = rows.reshape(*rows.shape[:-1], -1, 32)
    codes = np.zeros(blocks.shape, np.uint8)
    scales = np.zeros(blocks.shape[:-1], np.uint8)
    values = np.empty(blocks.shape)
    for at in np.ndindex(*blocks.shape[:-1]):
        x = blocks[at]
        if not np.isfinite(x).all():
            scales[at], values[at] = NAN, np.nan
            continue
        amax = np.abs(x).max()
        e = EXP_MIN
        if amax > 0:
            low = int(np.floor(np.log2(amax)))
            low += int(2.0 ** (low + 1) <= amax) - int(2.0 ** low > amax)
            e = min(max(low - 2 + (amax >= 1.75 * 2.0 ** low), EXP_MIN), EXP_MAX)
        unit = 2.0 ** e
        for i, v in enumerate(x):
            gap = np.abs(GRID - min(abs(v) / unit, 6.0))  # (past the largest code a gap would lose the grid in 64 bits)
            best = np.flatnonzero(gap == gap.min())
            place = best[0] if len(best) == 1 else best[best % 2 == 0][0]
            codes[at][i] = place | (8 if np.signbit(v) else 0)
            values[at][i] = np.copysign(GRID[place] * unit, v)
        scales[at] = e + 127
    return codes.reshape(rows.shape), scales, values.reshape(rows.shape)


class Tables:
    """Block tables over a stack of free pages, one page at a time."""

    def __init__(self, requests: int, width: int, pages: int, page: int, free=None):
        self.page, self.width = page, width
        self.free = list(range(pages - 1, -1, -1)) if free is None else list(free)
        self.table = [[] for _ in range(requests)]
        self.lengths = [0] * requests

    def pages_of(self, tokens: int) -> int:
        return -(-tokens // self.page)

    def assign(self, new, rows: int):
        """(slots, positions, cu, why it was refused or 0)."""
        new = [max(int(n), 0) for n in new]
        after = [self.pages_of(l + n) for l, n in zip(self.lengths, new)]
        need = sum(a - len(t) for a, t in zip(after, self.table))
        slots, positions = [-1] * rows, [-1] * rows
        refused = 1 if sum(new) > rows else 2 if max(after) > self.width else 3 if need > len(self.free) else 0
        if refused:
            return slots, positions, [0] * (len(new) + 1), refused
        cu = [0]
        for b, n in enumerate(new):
            while len(self.table[b]) < after[b]:
                self.table[b].append(self.free.pop())
            for i in range(n):
                at = self.lengths[b] + i
                slots[cu[b] + i] = self.table[b][at // self.page] * self.page + at % self.page
                positions[cu[b] + i] = at
            self.lengths[b] += n
            cu.append(cu[b] + n)
        return slots, positions, cu, 0

    def trim(self, keep) -> None:
        given = []
        for b, k in enumerate(keep):
            self.lengths[b] = min(self.lengths[b], max(int(k), 0))
            left = self.pages_of(self.lengths[b])
            given += self.table[b][left:]
            del self.table[b][left:]
        self.free += given[::-1]


def attend(query, keys, values, scaling: float, window: int | None = None):
    """Causal attention of the last len(query) tokens: query [n, Hq, D], keys and values [total, Hkv, D] -> [n, Hq, D]
    in float64; a row that sees no token is zero.  A token that a row does not see has no part in it, whatever it
    holds."""
    query, keys, values = (np.asarray(a, dtype=np.float64) for a in (query, keys, values))
    n, q_heads, _ = query.shape
    total, kv_heads, _ = keys.shape
    out = np.zeros(query.shape)
    for i in range(n):
        position = total - n + i
        first = 0 if window is None else max(0, position - window + 1)
        if position < first:
            continue
        for h in range(q_heads):
            kv = h // (q_heads // kv_heads)
            scores = keys[first:position + 1, kv] @ query[i, h] * scaling
            weights = np.exp(scores - scores.max())
            out[i, h] = (weights / weights.sum()) @ values[first:position + 1, kv]
    return out


def rotate(rows, positions, cos, sin, interleaved: bool = False):
    """Rows [n, H, D] rotated to their positions in float64: pair i of the first 2 * cos.shape[1] dimensions is i and
    i + cos.shape[1], or 2i and 2i + 1 if ``interleaved``; NaN where the tables have no row for a position."""
    rows = np.array(rows, dtype=np.float64)
    pairs = cos.shape[1]
    for t, position in enumerate(positions):
        if not 0 <= position < len(cos):
            rows[t] = np.nan
            continue
        for i in range(pairs):
            one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
            x, y = rows[t, :, one].copy(), rows[t, :, two].copy()
            c, s = float(cos[position, i]), float(sin[position, i])
            rows[t, :, one], rows[t, :, two] = x * c - y * s, y * c + x * s
    return rows


def attend_shaped(query, keys, values, scaling: float, window: int | None = None, cap: float | None = None, slopes=None,
                  sinks=None, first=None, last=None):
    """``attend`` of shaped scores: capped, less slopes[h] times the distance, beside a sink of sinks[h], over the tokens
    from first[i] to last[i] (0 and the row's own position by default) that there are."""
    query, keys, values = (np.asarray(a, dtype=np.float64) for a in (query, keys, values))
    n, q_heads, _ = query.shape
    total, kv_heads, _ = keys.shape
    out = np.zeros(query.shape)
    for i in range(n):
        position = total - n + i
        low = 0 if first is None else max(0, int(first[i]))
        if window is not None:
            low = max(low, position - window + 1)
        high = min(position if last is None else int(last[i]), total - 1)
        if high < low:
            continue
        at = np.arange(low, high + 1)
        for h in range(q_heads):
            kv = h // (q_heads // kv_heads)
            scores = keys[at, kv] @ query[i, h] * scaling
            if cap is not None:
                scores = cap * np.tanh(scores / cap)
            if slopes is not None:
                scores = scores - float(slopes[h]) * np.abs(position - at)
            top = scores.max() if sinks is None else max(scores.max(), float(sinks[h]))
            weights = np.exp(scores - top)
            whole = weights.sum() + (0.0 if sinks is None else np.exp(float(sinks[h]) - top))
            out[i, h] = (weights / whole) @ values[at, kv]
    return out
