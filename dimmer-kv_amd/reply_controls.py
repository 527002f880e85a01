"""Controls of a reply's logits: penalties for repeated tokens, biases and a grammar's masks, and the token picked, in one
pass over the logits (dkv_adjust_logits; include/dimmerkv.h states the arithmetic).

``ReplyControls`` holds the controls of a batch of replies on the GPU; ``apply`` takes the logits of a step and the
tokens so far.  ``greedy_answer(..., controls=...)`` answers under them.  Calls on one object, its copies and graphs captured
from them share words that their workgroups count on, and belong on one stream (or on streams the caller orders).
"""

from __future__ import annotations

import itertools

import torch

import dkv_hip

ARRIVAL_SETS = 256


def pack_allowed(mask: torch.Tensor) -> torch.Tensor:
    """bool [masks, vocab] -> int32 [masks, ceil(vocab / 32)], bit t % 32 of word t / 32 for token t."""
    masks, vocab = mask.shape
    bits = torch.nn.functional.pad(mask.to(torch.int64), (0, -vocab % 32)).view(masks, -1, 32)
    words = (bits << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


class ReplyControls:
    def __init__(self, rows: int, vocab: int, repetition=None, presence=None, frequency=None, bias=None, allowed=None,
                 device="cuda"):
        """Controls of ``rows`` replies over ``vocab`` tokens.

        - ``repetition`` (> 0; 1 is none) divides the positive and multiplies the other logits of tokens the history
          holds, ``presence`` and ``frequency`` are subtracted once and per occurrence in the reply: numbers, or float32
          [rows];
        - ``bias``: added to logits; {token: value} for every row, a list of such dicts by row, or (ids int32,
          values float32, cu int32 [rows + 1]); of an id that a row lists twice the last value counts;
        - ``allowed``: bool [rows, vocab] or [1, vocab] (every row), or (words int32 [masks, ceil(vocab / 32)],
          mask of each row int32 [rows], -1 for none; a number past the masks allows nothing).  ``allow`` changes it
          later.

        A captured ``apply`` reads the memory of its capture: bool masks given to ``allow`` later go into the memory of
        the first of their shape, so replays see them; words and mask numbers given as a tuple of GPU tensors are read
        where they are, and so are the values of biases: the caller may change them.  Which tokens of which rows have a
        bias is fixed here (ids and cu are copied: equal ids of a row are sorted out once)."""
        if rows < 0 or rows > 65535 or vocab < 1:
            raise ValueError(f"ReplyControls: {rows} rows (at most 65535) of {vocab} tokens")
        if torch.device(device).type != "cuda":
            raise ValueError("ReplyControls needs a GPU (the HIP path has no CPU fallback)")
        self.rows, self.vocab = rows, vocab
        self.device = torch.empty(0, device=device).device
        self._args = dkv_hip.LogitsArgs()
        self._args.rows, self._args.vocab = rows, vocab
        # words that a call's workgroups count themselves on (zero between calls); calls take turns over the sets, which
        # come round again: calls on one object are ordered
        self._arrivals = torch.zeros(ARRIVAL_SETS, max(rows, 1), dtype=torch.int32, device=device)
        start, step = self._arrivals.data_ptr(), self._arrivals.stride(0) * 4
        self._turns = itertools.cycle(range(start, start + ARRIVAL_SETS * step, step))
        self._held = {}  # the tensors whose addresses the arguments hold
        self._masks, self._first = {}, None  # words of bool masks by their number, and the row of zeros for a single one
        for name, value in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
            if value is not None:
                self._hold(name, self._per_row(name, value))
        if bias is not None:
            self._set_bias(bias)
        if allowed is not None:
            self.allow(allowed)

    def __copy__(self) -> "ReplyControls":
        """The same controls, with masks of its own from now on: bool masks given to one do not reach the other."""
        other = ReplyControls.__new__(ReplyControls)
        other.__dict__.update(self.__dict__)
        other._args = dkv_hip.LogitsArgs.from_buffer_copy(self._args)
        other._held, other._masks = dict(self._held), {}
        words = self._held.get("allowed")
        if any(words is kept for kept in self._masks.values()):
            other._hold("allowed", words.clone())
        return other

    def _hold(self, name: str, t: torch.Tensor) -> None:
        self._held[name] = t
        setattr(self._args, name, dkv_hip.ptr(t) if t.numel() else None)

    def _per_row(self, name: str, value) -> torch.Tensor:
        if not torch.is_tensor(value):
            if name == "repetition" and not value > 0:
                raise ValueError(f"ReplyControls: repetition {value} must be above 0")
            return torch.full((self.rows,), float(value), dtype=torch.float32, device=self.device)
        if value.shape != (self.rows,) or value.dtype != torch.float32:
            raise ValueError(f"ReplyControls: {name} must be a number or float32 [{self.rows}]")
        return value.to(self.device).contiguous()

    def _set_bias(self, bias) -> None:
        if not isinstance(bias, tuple):
            by_row = [bias] * self.rows if isinstance(bias, dict) else list(bias)
            if len(by_row) != self.rows:
                raise ValueError(f"ReplyControls: biases of {len(by_row)} rows, not {self.rows}")
            if any(not 0 <= token < self.vocab for row in by_row for token in row):
                raise ValueError(f"ReplyControls: biases of tokens outside 0..{self.vocab - 1}")
            cu = [0]
            for row in by_row:
                cu.append(cu[-1] + len(row))
            bias = (torch.tensor([token for row in by_row for token in row], dtype=torch.int32),
                    torch.tensor([value for row in by_row for value in row.values()], dtype=torch.float32),
                    torch.tensor(cu, dtype=torch.int32))
        ids, values, cu = bias
        if (ids.dtype != torch.int32 or values.dtype != torch.float32 or cu.dtype != torch.int32 or ids.dim() != 1
                or ids.shape != values.shape or cu.shape != (self.rows + 1,)):
            raise ValueError(f"ReplyControls: bias must be (int32 [n], float32 [n], int32 [{self.rows + 1}])")
        ids, values, cu = (t.to(self.device).contiguous() for t in (ids, values, cu))
        for name, t in (("bias_ids", self._last_of_each(ids, cu)), ("bias_values", values), ("bias_cu", cu.clone())):
            self._hold(name, t)
        self._args.biases = ids.shape[0]

    def _last_of_each(self, ids: torch.Tensor, cu: torch.Tensor) -> torch.Tensor:
        """The ids with -1 for all but a row's last mention of each: a stable sort by row and id puts that one last."""
        if ids.numel() == 0:
            return ids.clone()
        row = torch.searchsorted(cu, torch.arange(ids.numel(), dtype=torch.int32, device=self.device), right=True)
        key, place = torch.sort(row * (1 << 32) + ids, stable=True)
        last = torch.nn.functional.pad(key[1:] != key[:-1], (0, 1), value=True)
        return torch.empty_like(ids).scatter_(0, place, torch.where(last, ids[place], torch.full_like(ids, -1)))

    def allow(self, allowed) -> None:
        """The tokens that may be picked from now on (as ``allowed`` of the constructor, or None for all)."""
        if allowed is None:
            self._held.pop("allowed", None), self._held.pop("allowed_row", None)
            self._args.allowed = self._args.allowed_row = None
            return
        row = None
        if isinstance(allowed, tuple):
            words, row = allowed
        else:
            if allowed.dtype != torch.bool or allowed.dim() != 2 or allowed.shape[1] != self.vocab:
                raise ValueError(f"ReplyControls: allowed must be bool [rows, {self.vocab}] or (words, mask of each row)")
            words = pack_allowed(allowed)
            if allowed.shape[0] == 1:
                if self._first is None:
                    self._first = torch.zeros(self.rows, dtype=torch.int32, device=self.device)
                row = self._first
        need = -(-self.vocab // 32)
        if words.dtype != torch.int32 or words.dim() != 2 or words.shape[1] < need:
            raise ValueError(f"ReplyControls: mask words must be int32 [masks, {need}]")
        if row is None and words.shape[0] < self.rows:
            raise ValueError(f"ReplyControls: {words.shape[0]} masks for {self.rows} rows")
        if row is not None and (row.dtype != torch.int32 or row.shape != (self.rows,)):
            raise ValueError(f"ReplyControls: the mask of each row must be int32 [{self.rows}]")
        if not isinstance(allowed, tuple):  # into the words that captured calls may be reading
            held = self._masks.get(words.shape[0])
            words = self._masks.setdefault(words.shape[0], words.to(self.device)) if held is None else held.copy_(words)
        self._hold("allowed", words.to(self.device).contiguous())
        self._args.masks, self._args.words = words.shape
        self._args.allowed_row = None
        if row is not None:
            self._hold("allowed_row", row.to(self.device).contiguous())

    def apply(self, logits: torch.Tensor, tokens: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
              reply_start: torch.Tensor | None = None, out: torch.Tensor | None = None):
        """(adjusted logits, pick) of logits [rows, vocab] (float32, float16 or bfloat16).  Row r's history is the first
        ``lengths[r]`` of ``tokens`` [rows, history] (int64 or int32; all of them by default), its reply begins at
        ``reply_start[r]`` (0 by default).  ``out`` may be ``logits``, but not lie over other rows of them.  pick int64
        [rows] is the largest logit's token, the lowest of equals, -1 where no token is allowed.  No backward pass: asking
        a recorded call for its gradient raises."""
        if logits.device != self.device:
            raise ValueError(f"ReplyControls: logits must be on {self.device} (got {logits.device})")
        if tokens is not None and lengths is None:
            lengths = torch.full((self.rows,), tokens.shape[1], dtype=torch.int32, device=self.device)
        args = dkv_hip.LogitsArgs.from_buffer_copy(self._args)
        args.arrivals = next(self._turns)
        return dkv_hip.adjust_logits(args, logits, tokens, lengths, reply_start, out)


__all__ = ["ReplyControls", "pack_allowed"]
