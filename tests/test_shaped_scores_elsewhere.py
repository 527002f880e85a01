"""Recorded calls, contexts and places of shaped scores, on the CPU."""

from __future__ import annotations

import pytest
import torch

import dkv_hip
from test_paged_shaped_checks import rows_of, small_model


class Plain:
    """A context that says what scores it takes, and counts its calls."""

    def __init__(self, takes_shapes=None):
        self.calls = 0
        if takes_shapes is not None:
            self.takes_shapes = takes_shapes

    def attend(self, module, query, key, value, attention_mask, scaling):
        self.calls += 1
        return torch.zeros_like(query).transpose(1, 2), None


@pytest.mark.parametrize("family,words", [("Gemma2", "soft cap"), ("GptOss", "sinks")])
def test_contexts_of_plain_scores_refuse_others(family, words):
    """A context that attends by plain scores raises for a model whose scores are more, rather than answer by another formula;
    one that takes them, or does not say, is called."""
    import dimmer
    from compressed_attention import CompressedContext

    assert not CompressedContext.takes_shapes
    model = small_model(family)
    dimmer.install(model)
    ids = torch.randint(0, 50, (1, 7), generator=torch.Generator().manual_seed(1))
    for takes, refused in ((False, True), (True, False), (None, False)):
        context = Plain(takes)
        dimmer.STATE.compressed = context
        try:
            with torch.no_grad():
                if refused:
                    with pytest.raises(ValueError, match=words):
                        model(input_ids=ids)
                else:
                    model(input_ids=ids)
        finally:
            dimmer.STATE.compressed = None
        assert context.calls == (0 if refused else 2)


def test_a_plain_model_is_taken():
    """Models that hand the hook no cap and no sinks, or None for them, are served as before."""
    import dimmer

    context = Plain(False)
    module = torch.nn.Module()
    dimmer.STATE.compressed = context
    try:
        for more in ({}, dict(softcap=None), dict(s_aux=None, sliding_window=5)):
            dimmer.dimmer_attention(module, torch.zeros(1, 2, 3, 8), torch.zeros(1, 2, 3, 8), torch.zeros(1, 2, 3, 8), None, 1.0, **more)
    finally:
        dimmer.STATE.compressed = None
    assert context.calls == 3


def test_a_context_keeps_the_sinks_it_was_made_with():
    """As its documents say: sinks that are changed in place later are not the context's."""
    from paged_cache import PagedContext

    model = small_model("GptOss")
    shapes = PagedContext._layer_shapes(model, 2, "cpu")
    held = [shape["sinks"].clone() for shape in shapes]
    with torch.no_grad():
        for layer in model.model.layers:
            layer.self_attn.sinks.add_(1.0)
    assert all(torch.equal(shape["sinks"], was) for shape, was in zip(shapes, held))


def test_every_recorded_input_refuses_its_gradient():
    first, second, plain = torch.zeros(3, requires_grad=True), torch.zeros(3, requires_grad=True), torch.zeros(3)
    out = dkv_hip._recorded("this", torch.ones(3), first, None, plain, second)
    for t in (first, second):
        with pytest.raises(RuntimeError, match="this has no backward pass"):
            torch.autograd.grad(out.sum(), t, allow_unused=True, retain_graph=True)
    assert dkv_hip._recorded("this", plain, plain, None) is plain
    with torch.no_grad():
        assert not dkv_hip._recorded("this", torch.ones(3), first).requires_grad


def test_places_are_compared_on_the_host():
    """Whatever torch's default device is: a GPU's answer would have to be waited for, which a captured call may not."""
    storage = torch.zeros(4000)
    a, b = (rows_of(storage, at, 5, 3, 8, 40, 80) for at in (0, 16))
    args = dkv_hip.Fp4AttendArgs()
    args.query, args.query_token, args.query_head = b.data_ptr(), 40, 80
    out = rows_of(storage, 100, 5, 3, 8, 24, 8)

    def answers():
        return dkv_hip._rows_meet_rows(a, b), dkv_hip._query_meets(b, args, out), dkv_hip._rows_meet(0, 40, 16, 56, 5, 24)

    want = answers()
    with torch.device("meta"):
        assert answers() == want
