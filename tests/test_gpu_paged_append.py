"""Raw projections into the paged 4-bit cache, rotated on the way: codes and exponents equal to the oracle's of the exact
rotation, byte for byte, and queries rounded once (half a step of their type from the exact value)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_ref
from test_gpu_paged_attend import DEV, STEP, TYPES

pytestmark = pytest.mark.gpu
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}  # smallest steps


def tables(rows, pairs, base=10000.0):
    angle = np.arange(rows)[:, None] * base ** (-np.arange(pairs) / pairs)
    return (torch.tensor(f(angle), dtype=torch.float32, device=DEV) for f in (np.cos, np.sin))


def make(new, heads, dim, page=16, layers=1, rows=None, before=None):
    """A cache with tables in no order, and a step of ``new`` tokens after ``before``."""
    from paged_cache import PagedCache

    before = [0] * len(new) if before is None else before
    pages = sum(-(-(b + n) // page) for b, n in zip(before, new)) + 3
    cache = PagedCache(layers, heads, dim, pages, page=page, requests=len(new), device=DEV)
    cache.free.copy_(torch.randperm(pages, generator=torch.Generator().manual_seed(dim)).int())
    if any(before):
        cache.assign(before)
    step = cache.assign(new, rows)
    cache.check()
    return cache, step


def inputs(rows, q_heads, heads, dim, dtype, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    made = [torch.randn(rows, h, dim, generator=g, device=DEV) * s for h, s in ((q_heads, 1.5), (heads, 2.0), (heads, 1.0))]
    return [t.to(TYPES[dtype]) for t in made]


def near(got, exact, dtype):
    """Rounded once: within half a step."""
    got, dtype = got.double().cpu().numpy(), TYPES[dtype]
    return (np.abs(got - exact) <= STEP[dtype] * np.abs(exact) + TINY[dtype] / 2).all()


def check(cache, step, query, key, value, got, cos, sin, interleaved=False, layer=0):
    rows = [t.double().cpu().numpy() for t in (query, key, value)]
    positions = step.positions.tolist()
    kept = np.array([s >= 0 for s in step.slots.tolist()])
    cos, sin = cos.cpu().numpy(), sin.cpu().numpy()
    if got is not None:
        want = paged_ref.rotate(rows[0], positions, cos, sin, interleaved)
        assert near(got[torch.tensor(kept, device=DEV)], want[kept], {v: k for k, v in TYPES.items()}[query.dtype])
    held = [t.double().cpu().numpy() for t in cache.load(layer, step.slots, torch.float32)]
    for have, exact in zip(held, (paged_ref.rotate(rows[1], positions, cos, sin, interleaved), rows[2])):
        assert np.array_equal(have[kept], paged_ref.quantize(exact[kept])[2], equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 16), (64, 48), (128, 128), (128, 32), (128, 96), (256, 256), (256, 64)])
def test_shapes(dim, rotary, interleaved, dtype):
    cache, step = make([7, 0, 1, 30], 2, dim, before=[5, 3, 0, 100])
    query, key, value = inputs(step.rows, 6, 2, dim, dtype)
    cos, sin = tables(200, rotary // 2)
    got = cache.append(0, query, key, value, step, cos, sin, interleaved=interleaved)
    assert got.shape == query.shape and got.dtype == query.dtype
    check(cache, step, query, key, value, got, cos, sin, interleaved)
    place = query.clone()  # the queries' own
    assert cache.append(0, place, key, value, step, cos, sin, interleaved=interleaved, out=place) is place
    assert torch.equal(place, got)


@pytest.mark.parametrize("heads,q_heads", [(1, 1), (1, 7), (3, 3), (8, 32), (5, 40)])
@pytest.mark.parametrize("rows", [1, 2, 17, 64, 150])
def test_rows_and_heads(rows, heads, q_heads):
    cache, step = make([rows], heads, 128, page=32)
    query, key, value = inputs(rows, q_heads, heads, 128, "bf16", rows)
    cos, sin = tables(160, 64)
    check(cache, step, query, key, value, cache.append(0, query, key, value, step, cos, sin), cos, sin)


def test_large():
    """More rows than any launch shape's unit, in another layer; what stands before stays.  Against store of the rotated
    rows: the same bytes wherever float32 rows hold the exact rotation (no rotation at all)."""
    cache, step = make([5000, 1301], 4, 64, page=64, layers=2)
    query, key, value = inputs(step.rows, 8, 4, 64, "f16")
    cos, sin = tables(5000, 32)
    got = cache.append(1, query, key, value, step, cos, sin)
    some = torch.tensor([0, 1, 63, 64, 4999, 5000, 6300], device=DEV)
    from paged_cache import Step

    part = Step(step.slots[some], step.positions[some], step.cu, len(some), 1, 1)
    check(cache, part, query[some], key[some], value[some], got[some], cos, sin, layer=1)
    assert not cache.key_codes[0].any()
    cache.append(1, None, key, value, step, torch.ones_like(cos), torch.zeros_like(sin))
    held = [t.clone() for t in (cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales)]
    cache.store(0, key, value, step)
    for t in held:
        assert torch.equal(t[0] * 0 + t[1], t[1])
    for t, name in zip(held, ("key_codes", "key_scales", "value_codes", "value_scales")):
        assert torch.equal(getattr(cache, name)[0], t[1])


@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_and_the_queries_place(interleaved):
    """Views of one projection, heads before tokens, rows that are not aligned; the rotated queries in the place of the raw
    ones."""
    cache, step = make([40], 2, 64, layers=1)
    query, key, value = inputs(40, 4, 2, 64, "bf16")
    cos, sin = tables(40, 32)
    want = cache.append(0, query, key, value, step, cos, sin, interleaved=interleaved)
    codes = cache.key_codes.clone(), cache.value_codes.clone()

    def same(q, k, v, **more):
        for t in (cache.key_codes, cache.value_codes):
            t.zero_()
        got = cache.append(0, q, k, v, step, cos, sin, interleaved=interleaved, **more)
        assert torch.equal(got, want) and torch.equal(cache.key_codes, codes[0]) and torch.equal(cache.value_codes, codes[1])
        return got

    whole = torch.cat([t.flatten(1) for t in (query, key, value)], 1)
    parts = [t.unflatten(1, (-1, 64)) for t in whole.split([256, 128, 128], 1)]
    same(*parts)
    got = same(*parts, out=parts[0])
    assert got is parts[0] and torch.equal(whole[:, 256:384], key.flatten(1)) and torch.equal(whole[:, 384:], value.flatten(1))
    same(*(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (query, key, value)))
    same(*(torch.nn.functional.pad(t, (1, 0))[..., 1:] for t in (query, key, value)))
    out = torch.empty_like(query)
    assert same(query, key, value, out=out) is out
    wide = [torch.nn.functional.pad(t, (0, 32)) for t in (cos, sin)]  # halves of tables as models keep them
    cos, sin = (t[:, :32] for t in wide)
    same(query, key, value)


def test_padded_rows_and_positions_past_the_tables():
    """Rows behind the last request store nothing; their queries are zeros, or what the given out held.  A position that the
    tables lack makes its queries and keys NaN, and not its values."""
    cache, step = make([3, 2], 2, 64, rows=9, before=[30, 0])
    query, key, value = inputs(9, 4, 2, 64, "f32")
    cos, sin = tables(40, 32)
    got = cache.append(0, query, key, value, step, cos, sin)
    check(cache, step, query, key, value, got, cos, sin)
    assert not got[5:].any() and step.slots[5:].eq(-1).all()
    out = torch.full_like(query, 7.0)
    cache.append(0, query, key, value, step, cos, sin, out=out)
    assert torch.equal(out[:5], got[:5]) and (out[5:] == 7.0).all()
    cos, sin = cos[:32].contiguous(), sin[:32].contiguous()  # positions 30 and 31 are there, 32 is not
    got = cache.append(0, query, key, value, step, cos, sin)
    assert got[2].isnan().all() and got[[0, 1, 3, 4]].isfinite().all()
    keys, values = cache.load(0, step.slots, torch.float32)
    assert keys[2].isnan().all() and keys[[0, 1, 3, 4]].isfinite().all() and values.isfinite().all()
    check(cache, step, query, key, value, None, cos, sin)
    # a slot without a position: nothing can be rotated there
    step.positions[0] = -1
    got = cache.append(0, query, key, value, step, cos, sin)
    assert not got[0].any() and cache.load(0, step.slots[:1], torch.float32)[0].isnan().all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotations_next_to_a_border(interleaved):
    """Keys whose exact rotation lies between float32 numbers beside the border of two codes: x cos with a cosine of
    1 - 2^-24 is just below a tie for x on it, and a sine of 2^-20 times y of 2^-20 takes it past one by 2^-40."""
    cache, step = make([32], 1, 64)
    cos, sin = torch.full((32, 32), 1.0, device=DEV), torch.zeros(32, 32, device=DEV)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    one, two = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    key = torch.zeros(32, 1, 64)
    key[:, 0, one] = ties[torch.arange(32) % 7]
    key[:, 0, two] = torch.tensor([2.0 ** -20, -(2.0 ** -20)])[torch.arange(32) % 2]
    key[:, 0, one][:, 0] = 6.0  # the largest magnitude of the block: exponent 0
    key[:, 0, two][:, 0] = 6.0
    for c, s in ((1.0, 2.0 ** -20), (1.0 - 2.0 ** -24, 0.0), (1.0, 0.0), (1.0 - 2.0 ** -24, 2.0 ** -24), (1.0, 2.0 ** -30)):
        cos.fill_(c), sin.fill_(s)
        given = key.to(DEV)
        cache.append(0, None, given, given, step, cos, sin, interleaved=interleaved)
        check(cache, step, given, given, given, None, cos, sin, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_queries_are_rounded_once(interleaved, dtype):
    """Sums that a rounding to float32 on the way would take to a tie of the query's type, and off it to the wrong side."""
    cache, step = make([16], 1, 64)
    step_of = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}[dtype]
    one, two = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    query = torch.zeros(16, 1, 64, device=DEV)
    query[:, 0, one], query[:, 0, two] = 1.0 + step_of, 2.0 ** -14
    query = query.to(TYPES[dtype])
    for c, s in ((1.0, step_of * 2.0 ** 13), (1.0, -step_of * 2.0 ** 13), (1.0 - 2.0 ** -24, step_of * 2.0 ** 13), (1.0, 2.0 ** -30)):
        cos, sin = torch.full((16, 32), c, device=DEV), torch.full((16, 32), s, device=DEV)
        got = cache.append(0, query, query, query, step, cos, sin, interleaved=interleaved)
        want = paged_ref.rotate(query.double().cpu().numpy(), step.positions.tolist(), cos.cpu().numpy(), sin.cpu().numpy(), interleaved)
        assert torch.equal(got.double().cpu(), torch.tensor(want).to(TYPES[dtype]).double()) or dtype == "f32"
        assert near(got, want, dtype)


def test_infinities_nan_and_large_values():
    """A block that holds an infinity or a NaN once it is rotated is NaN; finite sums past float32 are the largest code."""
    cache, step = make([6], 1, 64)
    query, key, value = inputs(6, 2, 1, 64, "f32")
    key[0, 0, 3], key[1, 0, 40], key[2, 0, :] = float("inf"), float("nan"), 3.0e38
    query[0, 0, 3], query[1, 1, 40] = -float("inf"), float("nan")
    value[3, 0, 5], value[4, 0, 33] = float("inf"), 1e30
    cos, sin = tables(6, 32)
    cos[2], sin[2] = 0.9, -0.8
    got = cache.append(0, query, key, value, step, cos, sin)
    check(cache, step, query[2:], key, value, None, cos, sin)
    keys = cache.load(0, step.slots, torch.float32)[0]
    assert keys[0].isnan().all() and keys[1].isnan().all() and keys[2].abs().max() == 49152.0 and keys[2:].isfinite().all()
    bad = ~got.isfinite()
    assert bad[0, 0, [3, 35]].all() and bad[1, 1, [8, 40]].all() and bad.sum() == 4


def test_refusals():
    cache, step = make([5], 2, 64)
    query, key, value = inputs(5, 4, 2, 64, "f16")
    cos, sin = tables(8, 32)

    def refuse(words, q=query, k=key, v=value, c=cos, s=sin, **more):
        with pytest.raises(ValueError, match=words):
            cache.append(0, q, k, v, step, c, s, **more)

    refuse("key must be", k=key[:4])
    refuse("value must be", v=value.float())
    refuse("query must be", q=query.float())
    refuse("query must be", q=query[:, :, :32])
    refuse("cos must be", c=cos.double())
    refuse("cos must be", c=cos[:, 1:])
    refuse("sin must be", s=sin[:4])
    refuse("sin must be", s=sin.cpu())
    refuse("16-byte", c=cos.t().contiguous().t())
    refuse("multiple of 16", c=cos[:, :20], s=sin[:, :20])
    refuse("multiple of 16", c=torch.zeros(8, 40, device=DEV), s=torch.zeros(8, 40, device=DEV))
    refuse("out without queries", q=None, out=query)
    refuse("out must be", out=torch.empty(5, 4, 64, device=DEV))
    refuse("out must be", out=torch.empty(4, 5, 64, device=DEV, dtype=torch.float16).transpose(0, 1))
    room = torch.randn(9, 4, 64, device=DEV).half()
    refuse("lies over", q=room[:5], out=room[1:6])
    refuse("lies over", k=room[:5, :2], out=room[:5])
    refuse("lies over", v=room[:5, 2:], out=room[:5])
    refuse("lies over", q=room[:5, :2], k=room[:5, 1:3], out=room[:5, :2])
    refuse("lies over", q=room[:5, :1].expand(5, 4, 64), out=room[:5, :1].expand(5, 4, 64))
    with pytest.raises(ValueError, match="layer 1"):
        cache.append(1, query, key, value, step, cos, sin)
    assert not cache.key_codes.any()
    none = cache.assign([0])
    assert cache.append(0, query[:0], key[:0], value[:0], none, cos, sin).shape == (0, 4, 64)


@pytest.mark.parametrize("given", ["nothing", "the query's place"])
def test_recorded_calls_have_no_gradient(given):
    cache, step = make([5], 2, 64)
    query, key, value = inputs(5, 4, 2, 64, "f32")
    cos, sin = tables(8, 32)
    want = cache.append(0, query, key, value, step, cos, sin)
    assert not want.requires_grad
    leaf = query.clone().requires_grad_()
    rows = leaf * 1.0
    got = cache.append(0, rows, key, value, step, cos, sin, out=rows if given != "nothing" else None)
    assert got.requires_grad and torch.equal(got, want)
    with pytest.raises(RuntimeError, match="no backward pass"):
        got.sum().backward()
    held = leaf.detach().clone()
    with pytest.raises(RuntimeError, match="leaf"):
        cache.append(0, leaf, key, value, step, cos, sin, out=leaf)
    assert torch.equal(leaf, held)


def test_graph():
    """A captured step, replayed with other contents, equals the eager one."""
    cache, step = make([1, 1, 1], 2, 128, page=32, before=[100, 5, 31])
    query, key, value = inputs(3, 6, 2, 128, "bf16")
    cos, sin = tables(300, 64)
    new, keep = torch.ones(3, dtype=torch.int32, device=DEV), cache.lengths.clone()

    def body():
        step = cache.assign(new, 3, longest=300, most=1)
        return cache.append(0, query, key, value, step, cos, sin), step.slots

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        body()
        cache.trim(keep)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, slots = body()
    for turn in range(4):
        for t in (query, key, value):
            t.copy_(torch.randn_like(t))
        graph.replay()
        held = cache.load(0, slots, torch.float32)
        cache.trim(keep)
        torch.cuda.synchronize()
        want, at = body()
        cache.trim(keep)
        assert torch.equal(out, want) and torch.equal(at, slots), turn
        assert all(torch.equal(a, b) for a, b in zip(held, cache.load(0, at, torch.float32)))
        out.zero_()


@pytest.mark.parametrize("dim,rotary,interleaved", [(64, 64, False), (128, 64, True)])
def test_a_layer_as_it_serves(dim, rotary, interleaved):
    """Prompts, single tokens and a refused draft through append and attention of shaped scores: the answers are the
    formula's on the rotated rows the pages hold."""
    from paged_cache import PagedCache
    from test_gpu_paged_shaped import compare, numbers

    heads, groups = 2, 3
    cache = PagedCache(1, heads, dim, 40, page=16, requests=3, device=DEV)
    cos, sin = tables(256, rotary // 2)
    made = dict(cap=8.0, sinks=numbers(heads * groups, 1), window=60)
    g = torch.Generator(DEV).manual_seed(3)
    held = [[] for _ in range(3)]
    for new, keep in (([70, 0, 33], None), ([1, 1, 1], None), ([4, 4, 4], [2, 0, 4]), ([1, 40, 1], None), ([1, 1, 1], None)):
        step = cache.assign(new)
        whole = torch.randn(step.rows, (groups + 2) * heads * dim, generator=g, device=DEV).bfloat16()
        query, key, value = (t.unflatten(1, (-1, dim)) for t in whole.split([groups * heads * dim, heads * dim, heads * dim], 1))
        raw = key.double().cpu().numpy()
        turned = paged_ref.rotate(raw, step.positions.tolist(), cos.cpu().numpy(), sin.cpu().numpy(), interleaved)
        at = 0
        for b, n in enumerate(new):
            held[b] += list(turned[at:at + n])
            at += n
        query = cache.append(0, query, key, value, step, cos, sin, interleaved=interleaved, out=query)
        out = cache.attend_rows(0, query, step, **made)
        compare(cache, step, query, out, **made)
        if keep is not None:
            before = [len(h) - n for h, n in zip(held, new)]
            held = [h[:b + k] for h, b, k in zip(held, before, keep)]
            cache.trim([b + k for b, k in zip(before, keep)])
        cache.check()
    for b, rows in enumerate(held):
        keys = cache.load(0, cache.slots(b, 0, len(rows)), torch.float32)[0].double().cpu().numpy()
        assert np.array_equal(keys, paged_ref.quantize(np.stack(rows))[2])
