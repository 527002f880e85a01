"""Models whose scores are capped or joined by sinks behind the paged 4-bit cache (random weights, local configs): answers over
the pages against the same model attending, in 64 bits, to the values the pages hold."""

from __future__ import annotations

import pytest
import torch

from oracle import paged_ref
from test_gpu_model import _Tokenizer
from test_paged_shaped_checks import small_model

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Reference:
    """The context's attention by the oracle, on the values its cache holds once the new tokens are stored."""

    def __init__(self, context, model):
        self.context, self.model = context, model

    def attend(self, module, query, key, value, attention_mask, scaling):
        c, at = self.context, module.layer_idx
        c.attend(module, query, key, value, attention_mask, scaling)
        keys, values = (t.double().cpu().numpy() for t in c.cache.load(at, c.cache.slots(0, 0, c.tokens), torch.float32))
        config = self.model.config
        window = config.sliding_window if config.layer_types[at] == "sliding_attention" else None
        sinks = getattr(module, "sinks", None)
        out = paged_ref.attend_shaped(query[0].transpose(0, 1).double().cpu().numpy(), keys, values, scaling, window,
                                      cap=getattr(config, "attn_logit_softcapping", None),
                                      sinks=None if sinks is None else sinks.double().cpu().numpy())
        return torch.tensor(out, device=query.device).to(query.dtype).unsqueeze(0), None


@pytest.mark.parametrize("family", ["Gemma2", "GptOss"])
def test_answers_over_the_pages(family):
    import common
    import dimmer
    import methods
    from compressed_attention import greedy_answer
    from transformers import DynamicCache

    with torch.no_grad():
        model = small_model(family, window=100).to(DEV)
        dimmer.install(model)
        g = torch.Generator().manual_seed(2)
        ids, question = (torch.randint(0, 50, (1, n), generator=g).to(DEV) for n in (260, 9))
        past = model(input_ids=ids, past_key_values=DynamicCache(), use_cache=True).past_key_values
        keys, values = common.cache_tensors(past)
        assert keys[0].shape == keys[1].shape == (1, 2, 260, 64)
        context = methods.Methods("local", device=DEV, model=model).apply("fp4", keys, values, {}).stored
        text, logits = greedy_answer(model, _Tokenizer(), context, context.exact_cache, question, 260, max_new_tokens=6)
        context.rewind(260)
        want_text, want = greedy_answer(model, _Tokenizer(), Reference(context, model), context.exact_cache, question, 260,
                                        max_new_tokens=6)
        # two layers' attention in float32 against 64 bits: the hidden states agree to some 1e-6 of their size
        bound = 1e-4 * max(1.0, want.abs().max().item())
        assert text == want_text and (logits - want).abs().max() < bound
        # and the shapes matter: without them the logits are not the model's to that bound
        context.rewind(260)
        held, context._shapes = context._shapes, [{}, {}]
        _, plain = greedy_answer(model, _Tokenizer(), context, context.exact_cache, question, 260, max_new_tokens=1)
        assert (plain - want).abs().max() > bound
        context._shapes = held
        context.cache.check()
