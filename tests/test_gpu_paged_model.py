"""The paged 4-bit cache and the reply controls behind a Hugging Face Llama (random weights, local config): answers over
the pages against the same model attending, in 64 bits, to the values the pages hold."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import logits_ref, paged_ref
from test_gpu_model import _Tokenizer, _model_and_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield


class Reference:
    """The context's attention by the oracle, on the values its cache holds once the new tokens are stored."""

    def __init__(self, context):
        self.context = context

    def attend(self, module, query, key, value, attention_mask, scaling):
        c = self.context
        c.attend(module, query, key, value, attention_mask, scaling)
        keys, values = (t.double().cpu().numpy() for t in c.cache.load(module.layer_idx, c.cache.slots(0, 0, c.tokens), torch.float32))
        out = paged_ref.attend(query[0].transpose(0, 1).double().cpu().numpy(), keys, values, scaling)
        return torch.tensor(out, device=query.device).to(query.dtype).unsqueeze(0), None


def setup(tokens=300):
    import dimmer
    import methods

    model, keys, values, config = _model_and_cache(tokens, 5)
    dimmer.install(model)
    m = methods.Methods("local", device=DEV, model=model)
    g = torch.Generator("cpu").manual_seed(9)
    question = torch.randint(0, config.vocab_size, (1, 12), generator=g).to(DEV)
    return model, keys, values, m, question


def test_answers_over_the_pages():
    from compressed_attention import greedy_answer

    model, keys, values, m, question = setup()
    packed = m.apply("fp4", keys, values, {})
    context = packed.stored
    per_token = 2 * len(keys) * keys[0].shape[1] * 34  # 64 dimensions: 32 bytes of codes and 2 exponents
    assert packed.used_bytes == 300 * per_token and float(packed.token_bytes.sum()) == packed.used_bytes
    # the rebuilt caches hold the quantized rows
    for have, given in ((packed.keys[1], keys[1]), (packed.values[0], values[0])):
        want = paged_ref.quantize(given[0, :, :20].double().cpu().numpy())[2]
        assert np.array_equal(have[0, :, :20].double().cpu().numpy(), want) and have.shape == given.shape
    text, logits = greedy_answer(model, _Tokenizer(), context, context.exact_cache, question, 300, max_new_tokens=6)
    assert context.tokens == 300 + 12 + 5
    context.rewind(300)
    want_text, want = greedy_answer(model, _Tokenizer(), Reference(context), context.exact_cache, question, 300,
                                    max_new_tokens=6)
    # two layers' attention in float32 against 64 bits: the hidden states agree to some 1e-6, the logits are of order 10
    assert text == want_text and (logits - want).abs().max() < 1e-3
    context.rewind(300)
    again, _ = greedy_answer(model, _Tokenizer(), context, context.exact_cache, question, 300, max_new_tokens=6)
    assert again == text
    context.cache.check()


def test_context_refusals():
    from paged_cache import PagedContext

    model, keys, values, m, question = setup(40)
    context = PagedContext(keys, values, model, page=16, room=0)
    assert context.capacity == 48
    with pytest.raises(ValueError, match="pages for"):
        from compressed_attention import greedy_answer

        greedy_answer(model, _Tokenizer(), context, context.exact_cache, question, 40)
    with pytest.raises(ValueError):
        context.rewind(41)
    with pytest.raises(ValueError):
        PagedContext(keys, values[:1], model)
    with pytest.raises(ValueError, match="layer 1"):
        PagedContext([keys[0], keys[1][:, :, :30]], values, model)


def test_controlled_answers():
    """Replies under a repetition penalty, a bias and a grammar, each token the oracle's choice from the model's logits."""
    from compressed_attention import greedy_answer
    from reply_controls import ReplyControls

    model, keys, values, m, question = setup()
    vocab = model.config.vocab_size
    seen = []

    class Spy(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, *args, **kwargs):
            out = self.inner(*args, **kwargs)
            seen.append(out.logits[0, -1].float().cpu().numpy())
            return out

    def odd_after_even(reply):
        if not reply:
            return None
        mask = torch.zeros(vocab, dtype=torch.bool, device=DEV)
        mask[(1 - reply[-1] % 2)::2] = True
        return mask

    context = m.apply("fp4", keys, values, {}).stored
    past = torch.randint(0, vocab, (50,), device=DEV)
    controls = ReplyControls(1, vocab, repetition=1.5, presence=0.5, frequency=0.25, bias={3: 2.0, 8: -1.0})
    text, _ = greedy_answer(Spy(model), _Tokenizer(), context, context.exact_cache, question, 300, max_new_tokens=8,
                            controls=controls, history=past, grammar=odd_after_even)
    reply = [int(t) for t in text.split()]
    assert len(reply) == 8 and len(seen) == 8
    prompt = past.tolist() + question[0].tolist()
    for i, logits in enumerate(seen):
        mask = odd_after_even(reply[:i])
        _, want = logits_ref.adjust(logits, prompt + reply[:i], len(prompt), 1.5, 0.5, 0.25, [(3, 2.0), (8, -1.0)],
                                    None if mask is None else mask.cpu().numpy(), dtype=np.float32)
        assert reply[i] == want
    context.rewind(300)
    none = lambda reply: torch.zeros(vocab, dtype=torch.bool, device=DEV) if len(reply) == 2 else None
    text, _ = greedy_answer(model, _Tokenizer(), context, context.exact_cache, question, 300, max_new_tokens=8,
                            controls=ReplyControls(1, vocab), grammar=none)
    assert len(text.split()) == 2  # the grammar allows nothing more
    context.rewind(300)
    plain, _ = greedy_answer(model, _Tokenizer(), context, context.exact_cache, question, 300, max_new_tokens=4)
    context.rewind(300)
    free, _ = greedy_answer(model, _Tokenizer(), context, context.exact_cache, question, 300, max_new_tokens=4,
                            controls=ReplyControls(1, vocab))
    assert plain == free  # controls that change nothing choose as argmax does
    with pytest.raises(ValueError, match="grammar"):
        greedy_answer(model, _Tokenizer(), context, context.exact_cache, question, 300, grammar=none)


def test_serving_loop():
    """Requests that come, run and go over one cache, step by step: tables, stores, attention and picks against the
    oracle's, padding rows among them."""
    from paged_cache import PagedCache
    from reply_controls import ReplyControls

    requests, heads, groups, dim, page, layers, vocab = 4, 2, 2, 64, 16, 2, 300
    cache = PagedCache(layers, heads, dim, 24, page=page, requests=requests, table_pages=8, device=DEV)
    tables = paged_ref.Tables(requests, 8, 24, page)
    held = [[([], []) for _ in range(requests)] for _ in range(layers)]
    controls = ReplyControls(requests, vocab, repetition=1.3)
    tokens = torch.zeros(requests, 200, dtype=torch.int64, device=DEV)
    g = torch.Generator(DEV).manual_seed(3)
    plan = [([20, 0, 33, 1], None), ([1, 0, 1, 1], None), ([1, 17, 1, 1], [99, 99, 0, 99]), ([5, 1, 40, 1], [99] * 4),
            ([1, 1, 1, 0], [0, 10, 99, 99]), ([30, 1, 1, 9], None)]
    for new, keep in plan:
        rows = sum(new) + 2
        step = cache.assign(torch.tensor(new, dtype=torch.int32, device=DEV), rows, longest=128, most=max(new))
        slots, positions, cu, refused = tables.assign(new, rows)
        assert step.slots.tolist() == slots and step.cu.tolist() == cu and not refused
        for layer in range(layers):
            key, value = (torch.randn(rows, heads, dim, generator=g, device=DEV).bfloat16() for _ in range(2))
            query = torch.randn(rows, heads * groups, dim, generator=g, device=DEV).bfloat16()
            cache.store(layer, key, value, step)
            out = cache.attend_rows(layer, query, step)
            stored = [paged_ref.quantize(t.double().cpu().numpy())[2] for t in (key, value)]
            for b in range(requests):
                for x in range(2):
                    held[layer][b][x].extend(stored[x][cu[b]:cu[b + 1]])
                if new[b]:
                    want = paged_ref.attend(query[cu[b]:cu[b + 1]].double().cpu().numpy(), np.array(held[layer][b][0]),
                                            np.array(held[layer][b][1]), dim ** -0.5)
                    # the rounding of a bfloat16 of at most 8, and of the weights (2^-11) on values of at most 8
                    assert np.abs(out[cu[b]:cu[b + 1]].double().cpu().numpy() - want).max() < 8 * (2 ** -8 + 2 ** -10)
            assert not out[cu[-1]:].any()
        logits = torch.randn(requests, vocab, generator=g, device=DEV)
        _, pick = controls.apply(logits, tokens, cache.lengths, cache.lengths)
        for b in range(requests):
            _, want = logits_ref.adjust(logits[b].cpu().numpy(), tokens[b, :tables.lengths[b]].tolist(), tables.lengths[b],
                                        1.3, 0.0, 0.0, dtype=np.float32)
            assert int(pick[b]) == want
        tokens[torch.arange(requests, device=DEV), cache.lengths.long()] = pick
        if keep:
            cache.trim(keep)
            tables.trim(keep)
            for layer in range(layers):
                for b in range(requests):
                    for x in range(2):
                        del held[layer][b][x][tables.lengths[b]:]
    cache.check()


def test_grammar_ends_with_the_answer():
    """The masks that controls were made with hold again after an answer under a grammar."""
    from compressed_attention import greedy_answer
    from reply_controls import ReplyControls

    model, keys, values, m, question = setup()
    vocab = model.config.vocab_size
    context = m.apply("fp4", keys, values, {}).stored
    only = lambda token: torch.arange(vocab, device=DEV) == token
    controls = ReplyControls(1, vocab, allowed=only(7).unsqueeze(0))
    for grammar, want in ((None, "7 7"), (lambda reply: only(11), "11 11"), (None, "7 7"), (lambda reply: ~only(11) & only(11), ""),
                          (lambda reply: None, "%s"), (None, "7 7")):
        text, first = greedy_answer(model, _Tokenizer(), context, context.exact_cache, question, 300, max_new_tokens=2,
                                    controls=controls, grammar=grammar)
        assert text.split()[:1] == [str(int(first.argmax()))] if want == "%s" else text == want
        context.rewind(300)


def test_rebuilt_after_an_answer():
    """A compressed cache's keys and values are the prefill's, also when an answer lies behind them by then."""
    from compressed_attention import greedy_answer

    model, keys, values, m, question = setup()
    packed = m.apply("fp4", keys, values, {})
    greedy_answer(model, _Tokenizer(), packed.stored, packed.stored.exact_cache, question, 300, max_new_tokens=2)
    assert packed.stored.tokens == 313 and packed.token_bytes.shape == (300,)
    for have, given in ((packed.keys[0], keys[0]), (packed.values[1], values[1])):
        assert have.shape == given.shape
        want = paged_ref.quantize(given[0, :, 280:].double().cpu().numpy())[2]
        assert np.array_equal(have[0, :, 280:].double().cpu().numpy(), want)
    assert packed.stored.rebuilt()[0][0].shape[2] == 313


def test_sliding_window_layers():
    """Layers that the model's configuration gives a sliding window attend over it, the others over all tokens."""
    from types import SimpleNamespace

    from paged_cache import PagedContext
    from transformers import LlamaConfig

    heads, groups, dim, tokens, new, window = 2, 2, 64, 150, 20, 33
    shape = dict(num_hidden_layers=2, hidden_size=heads * groups * dim, num_attention_heads=heads * groups,
                 num_key_value_heads=heads, head_dim=dim)
    g = torch.Generator(DEV).manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    keys, values = ([rand(1, heads, tokens, dim) for _ in range(2)] for _ in range(2))
    config = LlamaConfig(sliding_window=window, layer_types=["full_attention", "sliding_attention"], **shape)
    context = PagedContext(keys, values, SimpleNamespace(config=config))
    for layer in range(2):
        module = SimpleNamespace(layer_idx=layer, num_key_value_groups=groups)
        query, key, value = rand(1, heads * groups, new, dim), rand(1, heads, new, dim), rand(1, heads, new, dim)
        have, _ = context.attend(module, query, *context.exact_cache.update(key, value, layer), None, dim ** -0.5)
        rows = [t.double().cpu().numpy() for t in context.cache.load(layer, context.cache.slots(0, 0, tokens + new), torch.float32)]
        want = paged_ref.attend(query[0].transpose(0, 1).double().cpu().numpy(), *rows, dim ** -0.5, window if layer else None)
        # float32 sums of at most 170 terms of order 1
        assert np.abs(have[0].double().cpu().numpy() - want).max() < 170 * 2.0 ** -22
    config = LlamaConfig(layer_types=["full_attention", "chunked_attention"], attention_chunk_size=64, **shape)
    with pytest.raises(ValueError, match="chunked"):
        PagedContext(keys, values, SimpleNamespace(config=config))


def test_a_forward_that_stops_half_way():
    """Tokens that some layers do not hold are not answered over: the next forward is refused until rewind forgets them."""
    from types import SimpleNamespace

    from paged_cache import PagedContext
    from transformers import LlamaConfig

    config = LlamaConfig(num_hidden_layers=3, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64)
    g = torch.Generator(DEV).manual_seed(6)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    keys, values = ([rand(1, 2, 30, 64) for _ in range(3)] for _ in range(2))
    context = PagedContext(keys, values, SimpleNamespace(config=config))

    def call(layer, new, broken=False):
        query, key, value = rand(1, 4, new, 64), rand(1, 2, new, 64), rand(1, 2, new, 64)
        module = SimpleNamespace(layer_idx=layer, num_key_value_groups=2)
        have, _ = context.attend(module, query, key[..., :32] if broken else key, value, None, 0.125)
        rows = [t.double().cpu().numpy() for t in context.cache.load(layer, context.cache.slots(0, 0, context.tokens), torch.float32)]
        want = paged_ref.attend(query[0].transpose(0, 1).double().cpu().numpy(), *rows, 0.125)
        # float32 sums of at most 40 terms of order 1
        assert np.abs(have[0].double().cpu().numpy() - want).max() < 40 * 2.0 ** -20
        assert rows[0].shape[0] == context.tokens

    for layer in range(3):
        call(layer, 3)
    with pytest.raises(ValueError, match="starts at layer 0"):
        call(1, 3)
    call(0, 3)
    with pytest.raises(ValueError, match=r"rewind\(33\)"):
        call(2, 3)  # a layer left out
    call(1, 3)
    for new in (3, 1):
        with pytest.raises(ValueError, match=r"rewind\(33\)"):
            call(0, new)
    context.rewind(33)
    assert context.tokens == 33
    with pytest.raises(ValueError):
        call(0, 2, broken=True)  # stopped inside its first layer
    with pytest.raises(ValueError, match=r"rewind\(33\)"):
        call(0, 1)
    for layer in range(3):  # tried again with as many tokens
        call(layer, 2)
    assert context.tokens == 35
    for layer in range(3):
        call(layer, 1)
    context.cache.check()
