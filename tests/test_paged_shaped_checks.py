"""What appending raw projections and attending with shaped scores refuse, before anything is launched (no GPU needed), and
their oracles against closed forms."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import dkv_hip
from oracle import paged_ref
from test_paged_cache_checks import P, attend_args, cache, refused


def append_args(**change):
    a = dkv_hip.Fp4AppendArgs()
    fields = dict(cache=cache(), query=P, key=P, value=P, out=P, query_token=256, query_head=64, key_token=128, key_head=64,
                  value_token=128, value_head=64, out_token=256, out_head=64, slots=P, positions=P, cos=P, sin=P, cos_row=32,
                  sin_row=32, table_rows=10, rotary=64, dtype=1, rows=5, q_heads=4)
    for name, value in (fields | change).items():
        setattr(a, name, value)
    return a


def append(a):
    return dkv_hip.lib().dkv_fp4_append(None if a is None else ctypes.addressof(a), None)


@pytest.mark.parametrize("change,code,words", [
    (dict(rotary=0), -2, "0 rotated"), (dict(rotary=24), -2, "24 rotated"), (dict(rotary=80), -2, "80 rotated"),
    (dict(rotary=-16), -2, "rotated"), (dict(table_rows=0), -2, "tables of 0"), (dict(q_heads=-1), -1, "-1 heads"),
    (dict(query=None), -1, "null queries"), (dict(q_heads=65533), -2, "65533 query heads"), (dict(dtype=3), -1, "dtype 3"),
    (dict(rows=-1), -2, "-1 rows"), (dict(rows=2**31 - 1), -2, "2147483647 rows"), (dict(key=None), -1, "null"),
    (dict(value=None), -1, "null"), (dict(slots=None), -1, "null"), (dict(positions=None), -1, "null"),
    (dict(cos=None), -1, "null"), (dict(sin=None), -1, "null"), (dict(out=None), -1, "null"), (dict(query=72), -1, "aligned"),
    (dict(out=72), -1, "aligned"), (dict(key=72), -1, "aligned"), (dict(cos=68), -1, "aligned"), (dict(sin=72), -1, "aligned"),
    (dict(key_token=124), -1, "multiples"), (dict(value_head=60), -1, "multiples"), (dict(query_head=60), -1, "multiples"),
    (dict(out_token=252), -1, "multiples"), (dict(cos_row=30), -1, "multiples"), (dict(cache=cache(head_dim=96)), -2, "head_dim")])
def test_append_refused(change, code, words):
    refused(append(append_args(**change)), code, words)


def test_append_of_nothing():
    refused(append(None), -1, "null arguments")
    assert append(append_args(rows=0)) == 0
    assert append(append_args(rows=0, key=None, cos=None, out=None)) == 0


def shape(**change):
    s = dkv_hip.Fp4Shape()
    for name, value in change.items():
        setattr(s, name, value)
    return s


@pytest.mark.parametrize("change,words", [
    (dict(cap=-1.0), "cap"), (dict(cap=float("nan")), "cap"), (dict(cap=float("inf")), "cap"), (dict(slopes=66), "misaligned"),
    (dict(sinks=65), "misaligned"), (dict(first=68), "misaligned"), (dict(last=68), "misaligned")])
def test_shapes_refused(change, words):
    lib, a, s = dkv_hip.lib(), attend_args(), shape(**change)
    refused(lib.dkv_fp4_attend_shaped(ctypes.addressof(a), ctypes.addressof(s), None, 0, None), -1, words)
    assert lib.dkv_fp4_attend_shaped_workspace_bytes(ctypes.addressof(a), ctypes.addressof(s)) == 0


@pytest.mark.parametrize("change,code,words", [
    (dict(q_heads=3), -2, "3 query heads"), (dict(window=-1), -2, "window"), (dict(query=None), -1, "null pointer"),
    (dict(table=None), -1, "null pointer"), (dict(query=72), -1, "aligned"), (dict(requests=0), -2, "bad shape")])
def test_shaped_calls_refused(change, code, words):
    lib, a, s = dkv_hip.lib(), attend_args(**change), shape(cap=2.0)
    need = lib.dkv_fp4_attend_shaped_workspace_bytes(ctypes.addressof(attend_args()), ctypes.addressof(s))
    assert need >= 16
    refused(lib.dkv_fp4_attend_shaped(ctypes.addressof(a), ctypes.addressof(s), P, 1 << 40, None), code, words)


def test_shaped_null_arguments_and_workspace():
    lib, a, s = dkv_hip.lib(), attend_args(longest=1 << 16, rows=1, most=1, requests=1), shape(cap=2.0)
    where, of = ctypes.addressof(a), ctypes.addressof(s)
    refused(lib.dkv_fp4_attend_shaped(None, of, None, 0, None), -1, "null arguments")
    refused(lib.dkv_fp4_attend_shaped(where, None, None, 0, None), -1, "null shape")
    none = attend_args(rows=0)
    assert lib.dkv_fp4_attend_shaped(ctypes.addressof(none), of, None, 0, None) == 0


def test_python_refusals():
    """On CPU tensors, and everything that is decided from shapes and types alone."""
    x, slots = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int64)
    table = torch.zeros(10, 32)
    with pytest.raises(ValueError, match="GPU"):
        dkv_hip.fp4_append(cache(), x, x, x, slots, slots, table, table)
    for bad in (dict(key=x[:2]), dict(value=x.half()), dict(slots=slots.int()), dict(positions=slots[:2])):
        given = dict(key=x, value=x, slots=slots, positions=slots) | bad
        with pytest.raises(ValueError):
            dkv_hip.fp4_append(cache(), x, given["key"], given["value"], given["slots"], given["positions"], table, table)
    for cap in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="cap"):
            dkv_hip._fp4_shape(0, 3, 4, cap, None, None, None, None)
    for at, wrong in ((0, torch.zeros(3)), (0, torch.zeros(4).double()), (1, torch.zeros(4, 1)), (2, torch.zeros(3).long()),
                      (3, torch.zeros(4).int())):
        given = [None] * 4
        given[at] = wrong
        with pytest.raises(ValueError, match="must be contiguous"):
            dkv_hip._fp4_shape(0, 3, 4, None, *given)


def rows_of(storage, offset, n, heads, dim, row, head):
    return torch.as_strided(storage, (n, heads, dim), (row, head, 1), offset)


def test_rows_that_share_memory():
    """Against a count of every element."""
    storage = torch.zeros(4000)
    g = np.random.RandomState(3)
    seen = {True: 0, False: 0}
    for _ in range(400):
        n, dim = int(g.randint(1, 6)), 8
        a, b = (rows_of(storage, int(g.randint(0, 60)) * 4, n, int(h), dim, int(g.choice([8, 16, 40, 64, 120])), int(g.choice([8, 12, 16, 80])))
                for h in g.randint(1, 4, 2))
        marks = []
        for t in (a, b):
            mark = torch.zeros_like(storage)
            index = torch.arange(4000)
            for place in torch.as_strided(index, t.shape, t.stride(), t.storage_offset()).reshape(-1, dim):
                mark[place] += 1
            marks.append(mark)
        meets = bool(((marks[0] > 0) & (marks[1] > 0)).any())
        if not dkv_hip._rows_lie_over(a):
            assert marks[0].max() == 1
            assert dkv_hip._rows_meet_rows(a, b) == meets
            seen[meets] += 1
        else:
            assert n > 1 or a.shape[1] > 1
    assert min(seen.values()) > 20
    fused = torch.zeros(7, 6 * 8)
    parts = [t.unflatten(1, (-1, 8)) for t in fused.split([24, 16, 8], 1)]
    assert not any(dkv_hip._rows_meet_rows(parts[i], parts[j]) for i in range(3) for j in range(3) if i != j)
    assert not dkv_hip._rows_lie_over(parts[0]) and dkv_hip._rows_lie_over(parts[2][:1].expand(7, 1, 8))


def test_oracle_rotation():
    """A quarter turn, both layouts; dimensions behind the rotated ones stay; the length of a pair does."""
    x = np.arange(1.0, 33.0).reshape(1, 1, 32)
    cos, sin = np.zeros((4, 8), np.float32), np.ones((4, 8), np.float32)
    half = paged_ref.rotate(x, [3], cos, sin)[0, 0]
    assert np.array_equal(half, np.concatenate([-x[0, 0, 8:16], x[0, 0, :8], x[0, 0, 16:]]))
    pairs = paged_ref.rotate(x, [3], cos, sin, interleaved=True)[0, 0]
    assert np.array_equal(pairs[:16], np.stack([-x[0, 0, 1:16:2], x[0, 0, 0:16:2]], -1).ravel())
    assert np.isnan(paged_ref.rotate(x, [4], cos, sin)).all()
    angle = np.random.RandomState(0).rand(4, 16)
    y = paged_ref.rotate(x, [2], np.cos(angle), np.sin(angle))[0, 0]
    assert np.allclose(np.hypot(y[:16], y[16:]), np.hypot(x[0, 0, :16], x[0, 0, 16:]))


def test_oracle_shaped_scores():
    rng = np.random.RandomState(1)
    query, keys, values = rng.randn(3, 4, 8), rng.randn(9, 2, 8), rng.randn(9, 2, 8)
    plain = paged_ref.attend(query, keys, values, 0.3, 4)
    assert np.allclose(paged_ref.attend_shaped(query, keys, values, 0.3, 4), plain)
    assert np.allclose(paged_ref.attend_shaped(query, keys, values, 0.3, 4, cap=1e7), plain)
    assert np.allclose(paged_ref.attend_shaped(query, keys, values, 0.3, 4, slopes=np.zeros(4), sinks=np.full(4, -np.inf)), plain)
    # a cap near 0 weighs every token the same; so does no scale, and a slope of log 2 halves a token's weight a step
    assert np.allclose(paged_ref.attend_shaped(query, keys, values, 0.3, cap=1e-9)[2], values.mean(0)[[0, 0, 1, 1]])
    weights = 0.5 ** np.arange(9)[::-1]
    falling = paged_ref.attend_shaped(query, keys, values, 0.0, slopes=np.full(4, np.log(2.0)))[2]
    assert np.allclose(falling, np.tensordot(weights / weights.sum(), values, 1)[[0, 0, 1, 1]])
    # a sink of score log 9 beside nine equal tokens takes half
    assert np.allclose(paged_ref.attend_shaped(query, keys, values, 0.0, sinks=np.full(4, np.log(9.0)))[2], values.mean(0)[[0, 0, 1, 1]] / 2)
    some = paged_ref.attend_shaped(query, keys, values, 0.0, first=[2, 5, -4], last=[4, 4, 100])
    assert np.allclose(some[0], values[2:5].mean(0)[[0, 0, 1, 1]]) and not some[1].any()
    assert np.allclose(some[2], values.mean(0)[[0, 0, 1, 1]])


def small_model(family, layers=2, window=None, seed=0):
    """A random model whose scores are capped (Gemma2), or joined by sinks (GptOss), with its sliding layers as they are."""
    import transformers

    torch.manual_seed(seed)
    sizes = dict(num_hidden_layers=layers, hidden_size=64, intermediate_size=64, num_attention_heads=4, num_key_value_heads=2,
                 head_dim=64, vocab_size=50, pad_token_id=0)
    if window:
        sizes |= dict(sliding_window=window)
    if family == "GptOss":
        sizes |= dict(num_local_experts=2, num_experts_per_tok=1)
    else:
        sizes |= dict(attn_logit_softcapping=3.0, query_pre_attn_scalar=16)
    model = getattr(transformers, f"{family}ForCausalLM")(getattr(transformers, f"{family}Config")(**sizes)).float().eval()
    with torch.no_grad():  # scores that reach the cap, and sinks that take their part
        for layer in model.model.layers:
            for projection in (layer.self_attn.q_proj, layer.self_attn.k_proj):
                projection.weight.mul_(8.0)
            if family == "GptOss":
                layer.self_attn.sinks.normal_(1.0, 2.0)
    return model


@pytest.mark.parametrize("family", ["Gemma2", "GptOss"])
def test_the_hook_keeps_caps_and_sinks(family):
    """The hook's own attention is the model's."""
    import dimmer

    model = small_model(family, window=16)
    ids = torch.randint(0, 50, (1, 40), generator=torch.Generator().manual_seed(1))
    model.set_attn_implementation("eager")
    with torch.no_grad():
        want = model(input_ids=ids).logits
    dimmer.install(model)
    with torch.no_grad():
        got = model(input_ids=ids).logits
    assert torch.allclose(got, want, atol=1e-5, rtol=1e-5), float((got - want).abs().max())


@pytest.mark.parametrize("family", ["Gemma2", "GptOss"])
def test_contexts_of_shaped_scores(family):
    """Such a model is taken with ``shaped`` (as far as the GPU that this test does without), each layer with its own shape."""
    from paged_cache import PagedContext

    model = small_model(family)
    caches = [torch.zeros(1, 2, 5, 64) for _ in range(2)]
    with pytest.raises(ValueError, match="soft cap|sinks"):
        PagedContext(caches, caches, model)
    with pytest.raises(ValueError, match="needs a GPU"):
        PagedContext(caches, caches, model, shaped=True)
    shapes = PagedContext._layer_shapes(model, 2, "cpu")
    if family == "Gemma2":
        assert shapes == [{"cap": 3.0}] * 2
    else:
        for shape, layer in zip(shapes, model.model.layers):
            assert list(shape) == ["sinks"] and torch.equal(shape["sinks"], layer.self_attn.sinks) and not shape["sinks"].requires_grad
        with pytest.raises(ValueError, match="sinks of layer 1"):
            PagedContext(caches[:1], caches[:1], model, shaped=True)
