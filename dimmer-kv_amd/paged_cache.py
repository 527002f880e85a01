"""A paged KV cache in 4 bits for many requests, attended to as it lies (MI355X HIP path).

Next to the calibrated codecs (kvtc.py, progressive.py), which compress a finished prefill, this cache needs no
calibration and grows while it serves: every new token's keys and values (RoPE applied) are quantized into pages, 32
dimensions to a power of two and 4 bits each (4.25 bits a value), and attention reads the pages.  include/dimmerkv.h
states the values, the pages' form and the tables.

``PagedCache`` holds the pages of every layer, the block tables and the free pages, all on the GPU; no call waits for
the GPU or reads from it, so a step can be captured in a HIP graph.  A step of a serving loop is

    step = cache.assign(new, rows)                    # pages, slots and positions of the step's tokens
    cache.store(layer, key, value, step)              # in every layer: the new rows into the pages,
    out = cache.attend_rows(layer, query, step)       # and the queries over all of them
    cache.trim(keep)                                  # finished requests, refused drafts

Calls on one cache share its tables and belong on one stream (or on streams the caller orders).

``PagedContext`` is the cache of one conversation behind a Hugging Face model: an attention context like
``CompressedContext`` (``dimmer.STATE.compressed``, ``greedy_answer``), whose new tokens go into the pages too.
"""

from __future__ import annotations

import itertools
from dataclasses import dataclass

import torch

import dkv_hip


@dataclass
class Step:
    """The rows of one step: requests one after another, ``cu`` the rows before each, -1 slots behind the last."""
    slots: torch.Tensor      # int64 [rows]
    positions: torch.Tensor  # int64 [rows]
    cu: torch.Tensor         # int32 [requests + 1]
    rows: int
    longest: int             # a bound on the requests' lengths, new tokens included: it shapes launches, not results
    most: int                # the same for the new tokens of a request


ARRIVAL_SETS = 256
ARRIVAL_WORDS = 256  # of a set: a launch that joins its splits has fewer than 512 workgroups, two of them at least a word
REFUSED = {1: "more new tokens than rows", 2: "a request passes its row of the block table", 3: "too few free pages"}


class PagedCache:
    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page: int = 64, requests: int = 1,
                 table_pages: int | None = None, device="cuda"):
        """``pages`` pages of ``page`` tokens (a power of two, 16 to 4096) in every layer, shared by ``requests``
        requests of at most ``table_pages`` pages each (all of them by default)."""
        table_pages = pages if table_pages is None else table_pages
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim {head_dim} is not 64, 128 or 256")
        if page < 16 or page > 4096 or page & (page - 1):
            raise ValueError(f"page {page} must be a power of two from 16 to 4096")
        if layers < 0 or kv_heads < 1 or pages < 1 or table_pages < 1 or not 1 <= requests <= 8192:
            raise ValueError(f"bad cache: {layers} layers, {kv_heads} KV heads, {pages} pages, {requests} requests of "
                             f"{table_pages} pages")
        if table_pages * page >= (1 << 31) - (1 << 16):
            raise ValueError(f"{table_pages} pages of {page} tokens pass 2^31 - 2^16 tokens a request")
        if torch.device(device).type != "cuda":
            raise ValueError("PagedCache needs a GPU (the HIP path has no CPU fallback)")
        self.layers, self.kv_heads, self.head_dim = layers, kv_heads, head_dim
        self.pages, self.page, self.requests, self.table_pages = pages, page, requests, table_pages

        def blank(width):
            return torch.zeros(layers, pages, kv_heads, page * width, dtype=torch.uint8, device=device)

        self.key_codes, self.value_codes = blank(head_dim // 2), blank(head_dim // 2)
        self.key_scales, self.value_scales = blank(head_dim // 32), blank(head_dim // 32)
        self.table = torch.full((requests, table_pages), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=device)
        self._state = torch.zeros(3, dtype=torch.int32, device=device)
        self.device = self.table.device
        self._pages = dkv_hip.Pages(self.lengths.data_ptr(), self.table.data_ptr(), self.free.data_ptr(),
                                    self.free_count.data_ptr(), self._state.data_ptr(), requests, table_pages, page, pages)
        self._layers = [dkv_hip.Fp4Cache(self.key_codes[i].data_ptr(), self.key_scales[i].data_ptr(),
                                         self.value_codes[i].data_ptr(), self.value_scales[i].data_ptr(), pages,
                                         kv_heads, page, head_dim) for i in range(layers)]
        # Words that the workgroups of one attention call count themselves on (zero between calls).  Calls take turns over
        # the sets, which come round again: calls on one cache are ordered, and the turns keep none apart for good.
        self._arrivals = torch.zeros(ARRIVAL_SETS, ARRIVAL_WORDS, dtype=torch.int32, device=device)
        start, step = self._arrivals.data_ptr(), ARRIVAL_WORDS * 4
        self._turns = itertools.cycle(range(start, start + ARRIVAL_SETS * step, step))
        self._attend = []
        for cache in self._layers:
            a = dkv_hip.Fp4AttendArgs()
            a.cache, a.table, a.lengths = cache, self.table.data_ptr(), self.lengths.data_ptr()
            a.requests, a.width, a.arrivals_count = requests, table_pages, ARRIVAL_WORDS
            self._attend.append(a)

    # ----- tables -----
    def _counts(self, counts, what: str) -> torch.Tensor:
        if not torch.is_tensor(counts):
            if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise ValueError(f"{what}: host numbers in a captured step, whose replays would read memory given back; it "
                                 "needs an int32 tensor on the GPU")
            return dkv_hip.to_device(list(counts), torch.int32, self.device)
        self._here(counts, what)
        return counts

    def assign(self, new, rows: int | None = None, longest: int | None = None, most: int | None = None) -> Step:
        """Pages for ``new`` tokens of each request (int32 [requests] on the GPU, as a captured step needs, or host numbers)
        and the slots and positions of the step's ``rows`` rows (needed with a GPU tensor; more than the new tokens for a padded step).
        ``longest`` and ``most`` bound the lengths and new tokens a request may have; they only shape later launches.
        If the pages, a table row or the rows do not suffice, nothing is assigned and every slot is -1; ``check``
        tells."""
        if not torch.is_tensor(new):
            new = [int(n) for n in new]
            rows = sum(max(n, 0) for n in new) if rows is None else rows
            most = max([0, *new]) if most is None else most
        if rows is None:
            raise ValueError("assign: a GPU tensor of new tokens needs rows, the step's number of rows")
        if not 0 <= rows < (1 << 31) - (1 << 16):
            raise ValueError(f"assign: {rows} rows")
        slots, positions = torch.empty(2, rows, dtype=torch.int64, device=self.device).unbind()
        step = Step(slots, positions, torch.empty(self.requests + 1, dtype=torch.int32, device=self.device), rows,
                    self.table_pages * self.page if longest is None else longest, rows if most is None else most)
        dkv_hip.page_assign(self._pages, self._counts(new, "assign"), rows, step.slots, step.positions, step.cu)
        return step

    def trim(self, keep) -> None:
        """Cut every request back to at most ``keep`` tokens (int32 [requests] on the GPU, as a captured step needs, or host
        numbers; 0 ends a request) and free the pages behind that."""
        dkv_hip.page_trim(self._pages, self._counts(keep, "trim"))

    def check(self) -> None:
        """Wait for the GPU and raise if the last ``assign`` or ``trim`` was refused."""
        state = self._state.tolist()
        if state[0]:
            raise dkv_hip.DkvError(f"assign: {REFUSED.get(state[0], state[0])}; nothing was assigned")
        if state[2]:
            raise dkv_hip.DkvError("trim: more pages given back than the cache has (a page in two requests?)")

    def slots(self, request: int, start: int, stop: int) -> torch.Tensor:
        """Slots int64 of tokens start..stop - 1 that a request holds."""
        if not 0 <= start <= stop <= self.table_pages * self.page:
            raise ValueError(f"slots: tokens {start} to {stop} of a request of at most {self.table_pages * self.page}")
        at = torch.arange(start, stop, device=self.device)
        return self.table[request].long()[at // self.page] * self.page + at % self.page

    # ----- rows -----
    def _layer(self, layer: int) -> dkv_hip.Fp4Cache:
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        return self._layers[layer]

    def _here(self, t: torch.Tensor, what: str) -> None:
        if t.device != self.device:
            raise ValueError(f"{what}: tensors must be on {self.device} (got {t.device})")

    def store(self, layer: int, key: torch.Tensor, value: torch.Tensor, step: Step) -> None:
        """The step's keys and values [rows, kv_heads, head_dim] (float32, float16 or bfloat16, any strides) into the
        pages of ``layer``; rows without a slot are left out."""
        self._here(step.slots, "store")
        dkv_hip.fp4_store(self._layer(layer), key, value, step.slots)

    def load(self, layer: int, slots: torch.Tensor, dtype: torch.dtype = torch.float16):
        """(keys, values) [n, kv_heads, head_dim] held in ``slots`` (int64 [n]); zeros for negative slots.  Every value
        is exact in the three types."""
        self._here(slots, "load")
        shape = (slots.shape[0], self.kv_heads, self.head_dim)
        key = torch.empty(shape, dtype=dtype, device=self.device)
        value = torch.empty_like(key)
        dkv_hip.fp4_load(self._layer(layer), slots, key, value)
        return key, value

    def attend_rows(self, layer: int, query: torch.Tensor, step: Step, scaling: float | None = None,
                    window: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the step's queries [rows, q_heads, head_dim] (float32, float16 or bfloat16, any strides) over
        the pages of ``layer``, where the step's own keys and values lie already: causal, and over the last ``window``
        tokens of each query's if given.  ``out`` (same shape and type, contiguous; it may be the query, but not lie over
        other rows of it) keeps its rows behind the last request; without it they are zeros.  No backward pass: asking a
        recorded call for its gradient raises."""
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        if query.dim() != 3 or query.shape[1] % self.kv_heads or query.shape[0] != step.rows:
            raise ValueError(f"attend_rows: query must be [{step.rows}, a multiple of {self.kv_heads}, {self.head_dim}] "
                             f"(got {list(query.shape)})")
        if window is not None and not 1 <= window < 1 << 31:
            raise ValueError(f"attend_rows: window {window}")
        self._here(step.cu, "attend_rows")
        args = dkv_hip.Fp4AttendArgs.from_buffer_copy(self._attend[layer])
        args.scaling = self.head_dim ** -0.5 if scaling is None else scaling
        args.window = window or 0
        args.arrivals = next(self._turns)
        args.longest, args.most = min(max(step.longest, 1), (1 << 31) - 1), min(max(step.most, 1), (1 << 31) - 1)
        return dkv_hip.fp4_attend(args, query, step.cu, out)

    def held_bytes(self) -> int:
        """GPU memory of the pages of all layers, the tables and the free list."""
        return sum(t.numel() * t.element_size() for t in (
            self.key_codes, self.key_scales, self.value_codes, self.value_scales, self.table, self.lengths, self.free,
            self.free_count, self._state, self._arrivals))


class PagedContext:
    """One conversation in a paged 4-bit cache, attended to directly: the ``attend`` contract of
    ``compressed_attention.CompressedContext`` for the ``dimmer`` hook.  Every forward's new keys and values are stored
    before they are attended to, in 4 bits as all others, so ``exact_cache`` (the cache the model updates) only carries
    them here: it starts empty.  Attention is causal, over all tokens or a layer's sliding window as the model's
    configuration has it; the model's additive mask is not read.  Models whose attention is more than that (a soft cap on
    scores, sinks beside the keys, other kinds of layers) are refused."""

    def __init__(self, keys: list[torch.Tensor], values: list[torch.Tensor], model, page: int = 64, room: int = 1024):
        """Per-layer [1, kv_heads, tokens, head_dim] keys (RoPE applied) and values on the GPU, with room for ``room`` more
        tokens."""
        first = keys[0]
        shape = first.shape
        if len(keys) != len(values) or len(shape) != 4 or shape[0] != 1:
            raise ValueError(f"PagedContext takes one conversation's per-layer [1, heads, tokens, head_dim] caches "
                             f"(got {len(keys)} and {len(values)} of {list(shape)})")
        if room < 0:
            raise ValueError(f"PagedContext: room {room}")
        self._windows = self._layer_windows(model.config, len(keys))
        self._refuse_more_than_scores(model)
        _, heads, tokens, dim = shape
        pages = max(1, -(-(tokens + room) // page))
        self.cache = PagedCache(len(keys), heads, dim, pages, page=page, device=first.device)
        self.capacity, self.tokens = pages * page, tokens
        self._model = model
        step = self.cache.assign([tokens], longest=tokens)
        for layer, (key, value) in enumerate(zip(keys, values)):
            if key.shape != shape or value.shape != shape:
                raise ValueError(f"layer {layer}: keys {list(key.shape)} and values {list(value.shape)}, not {list(shape)}")
            self.cache.store(layer, key[0].transpose(0, 1), value[0].transpose(0, 1), step)
        self._step, self._next = None, 0  # of the forward that runs: its rows, and the layer it is at
        self.exact_cache = self.fresh_cache()

    @staticmethod
    def _layer_windows(config, layers: int) -> list[int | None]:
        config = config.get_text_config(decoder=True)
        window = getattr(config, "sliding_window", None)
        kinds = getattr(config, "layer_types", None) or ["sliding_attention" if window else "full_attention"] * layers
        for kind in kinds:
            if kind not in ("full_attention", "sliding_attention"):
                raise ValueError(f"PagedContext: layers of {kind}")
        return [window if kind == "sliding_attention" else None for kind in kinds]

    @staticmethod
    def _refuse_more_than_scores(model) -> None:
        """Refuse models whose attention is not a softmax of scaled scores over the keys alone: the hook is given their
        soft cap (``softcap``) and sinks (``s_aux``), and would drop them."""
        if getattr(model.config.get_text_config(decoder=True), "attn_logit_softcapping", None):
            raise ValueError("PagedContext: the model's attention has a soft cap on its scores")
        if any(getattr(module, "sinks", None) is not None for module in getattr(model, "modules", tuple)()):
            raise ValueError("PagedContext: the model's attention has sinks beside its keys")

    def fresh_cache(self):
        """An empty cache for the model to update: one for every answer."""
        from transformers import DynamicCache

        return DynamicCache(config=self._model.config)

    def token_bytes(self) -> int:
        """Bytes of codes and exponents a token takes over all layers."""
        c = self.cache
        return 2 * c.layers * c.kv_heads * (c.head_dim // 2 + c.head_dim // 32)

    def rewind(self, tokens: int) -> None:
        """Forget everything behind the first ``tokens`` tokens (an answered question, say)."""
        if not 0 <= tokens <= self.tokens:
            raise ValueError(f"rewind to {tokens} of {self.tokens} tokens")
        self.cache.trim([tokens])
        self.tokens, self._step, self._next = tokens, None, 0
        self.exact_cache = self.fresh_cache()

    def rebuilt(self, dtype: torch.dtype = torch.float16, tokens: int | None = None):
        """(keys, values): per-layer [1, kv_heads, tokens, head_dim] caches of the values held, of the first ``tokens``
        if given."""
        slots = self.cache.slots(0, 0, self.tokens if tokens is None else min(tokens, self.tokens))
        rows = [self.cache.load(layer, slots, dtype) for layer in range(self.cache.layers)]
        return ([key.transpose(0, 1).contiguous().unsqueeze(0) for key, _ in rows],
                [value.transpose(0, 1).contiguous().unsqueeze(0) for _, value in rows])

    def attend(self, module, query, key, value, attention_mask, scaling):
        """Same contract as an HF attention function: returns (output [1, T, H, D], None).  A forward takes its layers in
        turn; after one that stopped half way ``rewind`` has to forget its tokens, which some layers do not hold."""
        layer, c = module.layer_idx, self.cache
        batch, q_heads, new, _ = query.shape
        if batch != 1:
            raise ValueError("PagedContext takes one conversation")
        if module.num_key_value_groups * c.kv_heads != q_heads:
            raise ValueError("module.num_key_value_groups does not match the cache's KV heads")
        if key is None or key.shape[2] < new:
            raise ValueError("PagedContext needs the new tokens' keys in the model's cache")
        if layer != self._next or (self._step is not None and self._step.rows != new):
            if self._step is None:
                raise ValueError("PagedContext: a forward starts at layer 0")
            raise ValueError(f"PagedContext: {new} tokens at layer {layer} where a forward of {self._step.rows} is at layer "
                             f"{self._next}; rewind({self.tokens - self._step.rows}) forgets one that stopped there")
        if self._step is None:  # a forward begins: pages for its tokens
            if self.tokens + new > self.capacity:
                raise ValueError(f"{self.tokens} + {new} tokens pass the {self.capacity} the context has pages for")
            self._step = c.assign([new], longest=self.tokens + new)
            self.tokens += new
        past = key.shape[2] - new
        c.store(layer, key[0, :, past:].transpose(0, 1), value[0, :, past:].transpose(0, 1), self._step)
        out = c.attend_rows(layer, query[0].transpose(0, 1), self._step, scaling=scaling, window=self._windows[layer])
        self._next = layer + 1
        if self._next == c.layers:
            self._step, self._next = None, 0
        return out.unsqueeze(0), None


__all__ = ["PagedCache", "PagedContext", "Step"]
