"""Logits of replies under penalties, biases and masks in numpy, token by token, in float32 as include/dimmerkv.h states
the operations (``dtype`` float32) or in 64 bits.  No counterpart in the reference."""

from __future__ import annotations

import numpy as np


def adjust(logits, history, reply_start, repetition, presence, frequency, bias=(), allowed=None, dtype=np.float64):
    """One row: logits [V], history a list of tokens, bias a list of (token, value), allowed bool [V] or None ->
    (adjusted [V], pick)."""
    x = np.array(logits, dtype=dtype)
    repetition, presence, frequency = dtype(repetition), dtype(presence), dtype(frequency)
    vocab = len(x)
    inside = [(i, int(t)) for i, t in enumerate(history) if 0 <= t < vocab]
    with np.errstate(all="ignore"):
        for t in {t for _, t in inside}:
            x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
            count = sum(1 for i, u in inside if u == t and i >= reply_start)
            if count:
                x[t] = x[t] - (frequency * dtype(count) + presence)
        for t, value in dict((t, v) for t, v in bias if 0 <= t < vocab).items():
            x[t] = x[t] + dtype(value)
    if allowed is not None:
        x[~np.asarray(allowed, dtype=bool)] = -np.inf
    if np.isnan(x).any():
        return x, int(np.flatnonzero(np.isnan(x))[0])
    return x, int(np.argmax(x)) if (x > -np.inf).any() else -1
