"""Compression methods by name: the entry points this package serves (the interface of
scripts/methods.py: ``Compressed``, ``budget_of``, ``Methods.codec`` / ``Methods.apply``, the
method-name mini-language and its error messages).

Served names (scripts/methods.py:1-33):

- ``full``: the uncompressed cache (control).
- ``fp4``: every token in 4 bits (paged_cache.PagedContext, 4.25 bits a value; no counterpart in the reference).  ``stored``
  is the context: ``greedy_answer(model, tokenizer, stored, stored.exact_cache, ...)`` answers over its pages; ``keys`` /
  ``values`` are rebuilt from them on first access.
- ``prog@<budget>[:snap][:r<frac>]``: progressive bit-plane kvtc with a hot tier of ``budget``
  and question-time refinement of the top ``frac`` tokens (scripts/methods.py:227-254).  The
  returned ``Compressed`` carries ``stored`` (the packed cache: ``stored.context(q_heads,
  exact_cache)`` answers directly over its codes on the GPU); ``refine`` follows the reference's
  closure (importance of the question over the hot tier, top ``frac`` middle tokens, cold planes
  fetched); ``keys``/``values`` are the hot tier rebuilt as FP16 caches, made on first access.
- ``kvtc@<budget>``, ``kvtcf@<budget>``, ``dkvtc@<budget>[:snap][:ev][:floor<x>][:kw<x>]``: kvtc
  transform coding with one rung or per-token rungs (scripts/methods.py:192-213,
  scripts/kvtc.py:157-274); answer over their codes with ``CompressedContext(codec, keys, values,
  model)``.

The uniform PCA / Lexico codecs and the H2O / dkv token allocators (scripts/methods.py:167-189,
:214-225) compress with other codecs and are not served here; naming them raises ``ValueError``.
"""

from __future__ import annotations

import time
from pathlib import Path

import torch

from kvtc import KVTCCodec
from progressive import ProgressiveCodec, importance_over_codes, question_importance

KVTC_PREFIXES = ("kvtc@", "kvtcf@", "dkvtc@")


class Compressed:
    """What ``Methods.apply`` returns (the fields of scripts/methods.py:52-63, plus ``stored``)."""

    def __init__(self, keys, values, evicted, used_bytes: int, seconds: float, histogram: dict | None = None,
                 refine=None, token_bytes: torch.Tensor | None = None, stored=None, rebuild=None):
        self._keys, self._values, self._rebuild = keys, values, rebuild
        self.evicted = evicted
        self.used_bytes = used_bytes
        self.seconds = seconds
        self.histogram = {} if histogram is None else histogram
        self.refine = refine            # refine(tail_ids, context_length) -> (keys, values, fetched bytes)
        self.token_bytes = token_bytes  # stored bytes per token (keys + values)
        self.stored = stored            # packed progressive cache (prog@)

    def _materialise(self):
        if self._keys is None and self._rebuild is not None:
            self._keys, self._values = self._rebuild()

    @property
    def keys(self):
        self._materialise()
        return self._keys

    @property
    def values(self):
        self._materialise()
        return self._values


def budget_of(name: str) -> float:
    """Nominal memory budget of a method name: 1.0 for ``full``, 4.25 of 16 bits for ``fp4``, the number after ``@`` (or after
    the first ``:`` of ``h2o:``/``dkv:`` names), NaN when the name implies none."""
    if name == "full":
        return 1.0
    if name == "fp4":
        return 4.25 / 16
    head, sep, rest = name.partition("@")
    if sep:
        return float(rest.split(":", 1)[0])
    if name.startswith(("h2o:", "dkv:")):
        return float(name.split(":")[1])
    return float("nan")


def synchronize(device) -> None:
    if torch.device(device).type == "cuda":
        torch.cuda.synchronize(device)


def _snap_weights(scores: dict) -> torch.Tensor:
    """Per-token importance: the SnapKV scores summed over layers and KV heads."""
    return torch.stack(scores["snap"]).sum(dim=(0, 1))


def _kvtc_plan(name: str, scores: dict) -> dict:
    """Options of a kvtc-family name; only ``dkvtc@`` takes :ev, :floor<x> and :kw<x>."""
    per_token = name.startswith("dkvtc@")
    budget, *options = name.split("@", 1)[1].split(":")
    plan = {"budget": float(budget), "per_token": per_token, "fill": name.startswith("kvtcf@"), "weights": None,
            "evict": False, "floor_share": 0.0, "key_weight": 1.0}
    for option in options:
        if option == "snap":
            plan["weights"] = _snap_weights(scores)
        elif per_token and option == "ev":
            plan["evict"] = True
        elif per_token and option.startswith("floor"):
            plan["floor_share"] = float(option[len("floor"):] or 0.5)
        elif per_token and option.startswith("kw"):
            plan["key_weight"] = float(option[len("kw"):])
        else:
            raise ValueError(f"Unknown option {option!r} in {name!r} "
                             "(dkvtc supports :snap, :ev, :floor, :kw<x>).")
    return plan


def _prog_plan(name: str, scores: dict) -> dict:
    budget, *options = name.split("@", 1)[1].split(":")
    plan = {"budget": float(budget), "weights": None, "fraction": 0.0}
    for option in options:
        if option == "snap":
            plan["weights"] = _snap_weights(scores)
        elif option.startswith("r"):
            plan["fraction"] = float(option[1:])
        else:
            raise ValueError(f"Unknown option {option!r} in {name!r}.")
    return plan


class Methods:
    """Applies named compression methods to a prefilled cache (scripts/methods.py:111-165)."""

    def __init__(self, model_id: str, basis=None, dictionary=None, device="cuda", recent: int = 32, model=None,
                 kvtc: str | Path | dict = "checkpoints/kvtc.pt",
                 progressive: str | Path | dict = "checkpoints/progressive.pt"):
        self.model_id = model_id
        self.device = device
        self.recent = recent
        self._model = model
        self._paths = {"kvtc": kvtc, "prog": progressive}
        self._codecs: dict[str, object] = {}

    def codec(self, kind: str):
        """The ``kvtc`` or ``prog`` codec, loaded on first use; refuses a calibration fit for
        another model."""
        if kind in self._codecs:
            return self._codecs[kind]
        if kind not in self._paths:
            raise ValueError(f"codec {kind!r} is not served by this package (kvtc and prog are)")
        if self._model is None:
            raise ValueError("kvtc methods need Methods(..., model=model) for RoPE tables.")
        source = self._paths[kind]
        if kind == "kvtc":
            loaded = KVTCCodec(source, self.device, self._model)
        else:
            loaded = ProgressiveCodec(self._paths["kvtc"], source, self.device, self._model)
        if loaded.model != self.model_id:
            label = kind if isinstance(source, dict) else source
            raise RuntimeError(f"{label} was fit for {loaded.model}; refit for {self.model_id}.")
        self._codecs[kind] = loaded
        return loaded

    def _timed(self, fn):
        synchronize(self.device)
        t0 = time.perf_counter()
        out = fn()
        synchronize(self.device)
        return out, time.perf_counter() - t0

    def apply(self, name: str, keys: list[torch.Tensor], values: list[torch.Tensor], scores: dict) -> Compressed:
        """Compress per-layer [1, kv_heads, tokens, head_dim] keys and values (scripts/methods.py:167-225)."""
        if name == "full":
            tokens = keys[0].shape[2]
            total = 2 * 2 * len(keys) * keys[0].numel()  # FP16 keys and values
            return Compressed(keys, values, None, total, 0.0,
                              token_bytes=torch.full((tokens,), total / tokens, device=self.device))
        if name == "fp4":
            return self._fp4(keys, values)
        if name.startswith("prog@"):
            return self._progressive(name, keys, values, scores)
        if name.startswith(KVTC_PREFIXES):
            return self._kvtc(name, keys, values, scores)
        raise ValueError(f"method {name!r} is not served by this package (full, fp4, prog@, kvtc@, kvtcf@, dkvtc@ are)")

    def _fp4(self, keys, values) -> Compressed:
        if self._model is None:
            raise ValueError("fp4 needs Methods(..., model=model) for the model's cache configuration.")
        from paged_cache import PagedContext

        stored, seconds = self._timed(lambda: PagedContext(keys, values, self._model))
        tokens, dtype = keys[0].shape[2], keys[0].dtype
        per_token = torch.full((tokens,), float(stored.token_bytes()), device=self.device)
        return Compressed(None, None, None, tokens * stored.token_bytes(), seconds, token_bytes=per_token, stored=stored,
                          rebuild=lambda: stored.rebuilt(dtype, tokens))

    def _kvtc(self, name: str, keys, values, scores) -> Compressed:
        plan = _kvtc_plan(name, scores)
        codec = self.codec("kvtc")
        result, seconds = self._timed(lambda: codec.compress(
            keys, values, plan["budget"], self.recent, plan["per_token"], fill=plan["fill"],
            weights=plan["weights"], evict=plan["evict"], floor_share=plan["floor_share"],
            key_weight=plan["key_weight"]))
        new_keys, new_values, used, histogram = result
        return Compressed(new_keys, new_values, codec.last_evicted, used, seconds, histogram,
                          token_bytes=self._kvtc_token_bytes(codec, keys[0].shape[2]))

    def _progressive(self, name: str, keys, values, scores) -> Compressed:
        plan = _prog_plan(name, scores)
        codec = self.codec("prog")
        tokens = keys[0].shape[2]
        fraction = plan["fraction"]
        # room in the hot blob for the tokens a question may refine
        expected_middle = max(0, tokens - min(codec.base.sinks, tokens) - self.recent)
        capacity = max(1, int(round(fraction * expected_middle))) if fraction > 0 else 0
        stored, seconds = self._timed(lambda: codec.encode(keys, values, plan["budget"], self.recent,
                                                           plan["weights"], refine_capacity=capacity))
        refine = self._refiner(stored, fraction) if fraction > 0 else None
        per_token = torch.full((tokens,), 2.0 * codec.exact_bytes, device=self.device)
        hot_sizes = [codec.orders[kind].prefix_bytes[store.hot_pieces].float() for kind, store in stored.stores.items()]
        per_token[stored.start:stored.end] = hot_sizes[0] + hot_sizes[1]
        return Compressed(None, None, None, stored.hot_bytes, seconds, refine=refine, token_bytes=per_token,
                          stored=stored, rebuild=stored.hot)

    @staticmethod
    def _top(scores: torch.Tensor, count: int) -> torch.Tensor:
        """Indices of the ``count`` largest ``scores`` (``importance.topk(count)``,
        scripts/methods.py:246-247): on the GPU the HIP radix select (dkv_topk, K4b), in ascending
        index order with ties to the lower index; torch's topk for CPU tensors.  The refine steps
        take the indices as a set, so the order does not matter."""
        if not scores.is_cuda:
            return scores.topk(count).indices
        import dkv_hip

        idx = torch.empty(count, dtype=torch.int32, device=scores.device)
        dkv_hip.topk(scores.float().contiguous(), count, idx)
        return idx.long()

    def _refiner(self, stored, fraction: float):
        """The question-time refinement closure (scripts/methods.py:244-248)."""
        middle = stored.end - stored.start
        count = max(1, int(round(fraction * middle)))

        def refine(tail_ids, context_length, exact_cache=None):
            """Importance of the question over the hot tier, top ``fraction`` middle tokens, cold
            planes fetched.  With ``exact_cache`` (sinks + recent window) the question runs over
            the codes and only the codes are refined (returns (None, None, fetched)); without it,
            over the rebuilt FP16 hot cache, returning the refined caches as the reference does."""
            if exact_cache is not None:
                context = stored.context(self._model.config.num_attention_heads, exact_cache)
                importance = importance_over_codes(self._model, context, exact_cache, tail_ids, context_length)
                return None, None, stored.refine_codes(self._top(importance, count) + stored.start)
            hot_keys, hot_values = stored.hot()
            importance = question_importance(self._model, hot_keys, hot_values, tail_ids, context_length)
            top = self._top(importance[stored.start:stored.end], count) + stored.start
            return stored.refine(hot_keys, hot_values, top)

        return refine

    def _kvtc_token_bytes(self, codec, tokens: int) -> torch.Tensor:
        """Bytes kept per token (keys + values) from the codec's last rung choice (scripts/methods.py:256-267):
        exact tokens at their FP16 size, compressed tokens at their rungs' sizes, evicted ones at 0."""
        start = min(codec.sinks, tokens)
        middle = codec.last_choice["key"].shape[0]
        kept = torch.zeros(middle, device=self.device)
        for kind, choice in codec.last_choice.items():
            sizes = torch.tensor(codec.streams[kind].rung_bytes + [codec.exact_bytes], dtype=torch.float32,
                                 device=self.device)
            kept += torch.where(choice >= 0, sizes[choice.clamp_min(0)], torch.zeros_like(kept))
        per_token = torch.full((tokens,), 2.0 * codec.exact_bytes, device=self.device)
        per_token[start:start + middle] = kept
        return per_token


__all__ = ["Compressed", "Methods", "budget_of", "synchronize"]
