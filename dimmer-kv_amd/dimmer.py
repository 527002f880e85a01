"""The ``dimmer`` attention hook for Hugging Face models (the answer-path interface of
scripts/dimmer.py: ``STATE`` :24-35, ``dimmer_attention`` :45-77, ``install`` :80-84,
``set_eviction`` :87-88, ``prefill_with_scores`` :91-121, ``mean_scores`` :124-129).

With ``STATE.compressed`` set (a ``CompressedContext``), every attention call of the model goes to
``CompressedContext.attend``, which runs the HIP kernels over the packed codes; this is the
dispatch the reference makes at scripts/dimmer.py:47-48.  A context whose ``takes_shapes`` is false
attends by plain scores, and calls of a model that caps them or has sinks raise.  Without it the hook is ordinary eager
attention over the cache the model holds, with the reference's two side duties: hiding evicted
(layer, KV head, token) slots, and recording the attention each token receives (the H2O sum over
all queries and the SnapKV sum over the last ``window`` queries) while ``STATE.scoring`` is on.
The Lexico allocator of scripts/dimmer.py:132-293 is an ablation and is not served here.
"""

from __future__ import annotations

import contextlib

import torch
import torch.nn.functional as F

ATTENTION_NAME = "dimmer"


class _State:
    """Module-wide hook state: score capture switches and buffers, eviction masks, and the
    compressed context answering in place of the cache."""

    def __init__(self):
        self.scoring = False
        self.window = 32
        self.scores: dict = {}         # layer -> [kv_heads, keys] attention received from every query
        self.window_scores: dict = {}  # layer -> [kv_heads, keys] from the last ``window`` queries
        self.evicted: dict = {}        # layer -> [kv_heads, context tokens], True = hidden
        self.compressed = None         # compressed_attention.CompressedContext or None


STATE = _State()


def _per_kv_head(received: torch.Tensor, groups: int) -> torch.Tensor:
    """[q_heads, keys] -> [kv_heads, keys]: sum over the query heads that share a KV head."""
    return received.unflatten(0, (-1, groups)).sum(dim=1)


def dimmer_attention(module, query, key, value, attention_mask, scaling, dropout=0.0, **kwargs):
    """HF attention function: ``query`` [B, q_heads, q, D], ``key``/``value`` [B, kv_heads, k, D];
    returns (output [B, q, q_heads, D], None) (scripts/dimmer.py:45-77)."""
    cap, sinks = kwargs.get("softcap"), kwargs.get("s_aux")  # of models that have them
    if STATE.compressed is not None:
        if not getattr(STATE.compressed, "takes_shapes", True) and (cap is not None or sinks is not None):
            raise ValueError(f"{type(STATE.compressed).__name__}: the model's attention has "
                             f"{'a soft cap on its scores' if cap is not None else 'sinks beside its keys'}, and the context's has not")
        return STATE.compressed.attend(module, query, key, value, attention_mask, scaling)
    groups = module.num_key_value_groups
    # query head h reads KV head h // groups; the key operand is made contiguous before the product
    keys_t = key.repeat_interleave(groups, dim=1).transpose(-1, -2).contiguous()
    logits = torch.matmul(query, keys_t).mul_(scaling)
    if cap is not None:
        logits = torch.tanh(logits / cap) * cap
    if attention_mask is not None:
        logits = logits + attention_mask
    evicted = STATE.evicted.get(module.layer_idx)
    if evicted is not None:
        # tokens appended after the context (the question, the reply) are never hidden
        hidden = F.pad(evicted.repeat_interleave(groups, dim=0), (0, logits.shape[-1] - evicted.shape[1]))
        logits = logits.masked_fill(hidden[None, :, None, :], torch.finfo(logits.dtype).min)
    if sinks is not None:
        logits = torch.cat([logits, sinks.to(logits.dtype).view(1, -1, 1, 1).expand(*logits.shape[:3], 1)], dim=-1)
    probs = torch.softmax(logits, dim=-1, dtype=torch.float32)
    if sinks is not None:
        probs = probs[..., :-1]
    if STATE.scoring:
        layer = module.layer_idx
        received = _per_kv_head(probs[0].sum(dim=1), groups)
        earlier = STATE.scores.get(layer)
        if earlier is not None:  # chunked prefill: this chunk's queries add to the earlier sums
            received[:, : earlier.shape[1]] += earlier
        STATE.scores[layer] = received
        # the last chunk always holds the whole window, so it overwrites earlier chunks' values
        STATE.window_scores[layer] = _per_kv_head(probs[0, :, -STATE.window:].sum(dim=1), groups)
    out = torch.matmul(probs.to(query.dtype), value.repeat_interleave(groups, dim=1))
    return out.transpose(1, 2).contiguous(), None


def install(model) -> None:
    """Register ``dimmer_attention`` (with HF's eager mask builder) and select it for ``model``."""
    from transformers import AttentionInterface
    from transformers.masking_utils import AttentionMaskInterface, eager_mask

    AttentionInterface.register(ATTENTION_NAME, dimmer_attention)
    AttentionMaskInterface.register(ATTENTION_NAME, eager_mask)
    model.set_attn_implementation(ATTENTION_NAME)


def set_eviction(evicted) -> None:
    """Per-layer [kv_heads, tokens] masks of hidden slots, or None to hide nothing."""
    STATE.evicted = {} if evicted is None else {layer: mask for layer, mask in enumerate(evicted)}


@contextlib.contextmanager
def recording(evicted=None):
    """Score capture around one or more forward passes: yields the per-layer dict
    ``{layer: [kv_heads, keys]}`` that fills with the attention each key receives (summed over the
    queries and the query heads of its KV head), with ``evicted`` slots hidden meanwhile."""
    set_eviction(evicted)
    STATE.scores, STATE.window_scores, STATE.scoring = {}, {}, True
    try:
        yield STATE.scores
    finally:
        STATE.scoring = False
        set_eviction(None)


def _chunk_bounds(tokens: int, chunk: int, window: int) -> list[int]:
    """Chunk edges 0 = e0 < e1 < ... = tokens; a last chunk shorter than ``window`` is merged into
    the one before it so the SnapKV window lies inside a single chunk."""
    edges = list(range(0, tokens, chunk)) + [tokens]
    if len(edges) > 2 and tokens - edges[-2] < window:
        del edges[-2]
    return edges


def prefill_with_scores(model, input_ids: torch.Tensor, window: int = 32, chunk: int = 512):
    """Chunked prefill of ``input_ids`` [1, tokens] through the hook (installed on ``model``) with
    score capture on; returns (cache, {"sum": [...], "snap": [...]}), per-layer [kv_heads, tokens]
    (scripts/dimmer.py:91-121).  ``scores["snap"]`` is what ``:snap`` method options weight by."""
    set_eviction(None)
    STATE.scores, STATE.window_scores, STATE.window, STATE.scoring = {}, {}, window, True
    edges = _chunk_bounds(input_ids.shape[1], chunk, window)
    cache = None
    try:
        for lo, hi in zip(edges, edges[1:]):
            positions = torch.arange(lo, hi, device=input_ids.device).unsqueeze(0)
            cache = model(input_ids=input_ids[:, lo:hi], past_key_values=cache, position_ids=positions,
                          use_cache=True).past_key_values
    finally:
        STATE.scoring = False
    layers = sorted(STATE.scores)
    return cache, {"sum": [STATE.scores[l] for l in layers], "snap": [STATE.window_scores[l] for l in layers]}


def mean_scores(scores: list[torch.Tensor]) -> list[torch.Tensor]:
    """Each token's summed score divided by the number of causal queries that can see it
    (``tokens - position``), removing the bias of sums toward early tokens."""
    tokens = scores[0].shape[-1]
    seen_by = tokens - torch.arange(tokens, device=scores[0].device, dtype=torch.float32)
    return [s / seen_by for s in scores]
