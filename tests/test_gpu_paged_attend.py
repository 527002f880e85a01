"""Attention over the paged 4-bit cache against oracle/paged_ref.attend in 64 bits on the values the cache holds.

A result may be off by the rounding of its type, u |ref|, and by an error of the weights p times what they weigh,
A = sum p |v|.  The weights' relative error: 2^-11 for their float16 rounding (2^-22 in two pieces for float32), twice
the error of a score (once above and once below the fraction line), and of the sums over n tokens, n 2^-24 at the most.
A score's error: D + 8 roundings of float32 on sum |q k| scaling, and of the exponent's argument, |score| + 16 in
units of 2^-24, with two units of the hardware's exponential.  A small weight is a subnormal float16, off by half of
2^-24 of what it is held in: 2^15 times for float32 against the largest weight, so 2^-40 sum |v| more; 2^8 times for
16-bit types against a reference that the largest weight may pass but not stay below, so 2^-33 sum |v|."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
WEIGHT = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -11}


def build(lengths, new, heads, dim, page, seed=0, spread=1.0, layers=1, room=0):
    """A cache whose requests hold ``lengths`` tokens before a step of ``new`` tokens each, and the step; ``room`` more
    pages for each request."""
    from paged_cache import PagedCache

    pages = sum(-(-(l + n) // page) for l, n in zip(lengths, new)) + room * len(lengths) + 2
    width = max(-(-(l + n) // page) for l, n in zip(lengths, new)) + room + 1
    cache = PagedCache(layers, heads, dim, pages, page=page, requests=len(lengths), table_pages=width, device=DEV)
    # free pages in no order, so that tables are none either
    cache.free.copy_(torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int())
    g = torch.Generator(DEV).manual_seed(seed)
    for counts in (lengths, new):
        step = cache.assign(counts, longest=max(l + n for l, n in zip(lengths, new)))
        if step.rows:
            rows = [torch.randn(step.rows, heads, dim, generator=g, device=DEV) * s for s in (spread, 1.0)]
            cache.store(layers - 1, rows[0], rows[1], step)
    cache.check()
    return cache, step


def compare(cache, step, query, got, scaling, window=None, layer=0):
    lengths, cu, dtype = cache.lengths.tolist(), step.cu.tolist(), query.dtype
    for b, total in enumerate(lengths):
        lo, hi = cu[b], cu[b + 1]
        if lo == hi:
            continue
        keys, values = (t.double().cpu().numpy() for t in cache.load(layer, cache.slots(b, 0, total), torch.float32))
        q = query[lo:hi].double().cpu().numpy()
        have = got[lo:hi].double().cpu().numpy()
        want = paged_ref.attend(q, keys, values, scaling, window)
        heads, groups = keys.shape[1], q.shape[1] // keys.shape[1]
        for i in range(hi - lo):
            at = total - (hi - lo) + i
            first = 0 if window is None else max(0, at - window + 1)
            for h in range(q.shape[1]):
                if at < first:
                    assert not have[i, h].any()
                    continue
                k, v = keys[first:at + 1, h // groups], values[first:at + 1, h // groups]
                score = k @ q[i, h] * scaling
                size = np.abs(k) @ np.abs(q[i, h]) * abs(scaling)
                p = np.exp(score - score.max())
                p /= p.sum()
                a = p @ np.abs(v)
                off = 2.0 ** -24 * ((k.shape[1] + 8) * size.max() + 2 * np.abs(score).max() + 32)
                weight = WEIGHT[dtype] + 2 * off + len(p) * 2.0 ** -24
                error = np.abs(have[i, h] - want[i, h])
                small = (2.0 ** -40 if dtype == torch.float32 else 2.0 ** -33) * np.abs(v).sum(0)
                assert (error <= STEP[dtype] * np.abs(want[i, h]) + weight * a + small).all(), (b, i, h, error.max())


def run(lengths, new, heads=2, groups=3, dim=64, page=16, dtype="bf16", window=None, scaling=None, spread=1.0, seed=0):
    print(f"[case] attend {lengths} + {new} heads={heads}x{groups} dim={dim} page={page} {dtype} window={window}", flush=True)
    cache, step = build(lengths, new, heads, dim, page, seed, spread)
    g = torch.Generator(DEV).manual_seed(seed + 1)
    query = (torch.randn(step.rows, heads * groups, dim, generator=g, device=DEV) * 1.5).to(TYPES[dtype])
    got = cache.attend_rows(0, query, step, scaling=scaling, window=window)
    assert got.shape == query.shape and got.dtype == query.dtype
    compare(cache, step, query, got, dim ** -0.5 if scaling is None else scaling, window)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32)])
def test_single_tokens(dim, page, dtype):
    """Lengths of one token, around a tile, a chunk, a page and a split."""
    run([0, 1, 14, 15, 16, 47, 62, 63, 64, 65, 200, 255, 256, 700], [1] * 14, dim=dim, page=page, dtype=dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,groups", [(1, 1), (3, 1), (8, 4), (2, 7), (1, 16), (1, 20), (2, 40)])
def test_heads(heads, groups, dtype):
    run([130, 3], [1, 1], heads=heads, groups=groups, dim=128, page=32, dtype=dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [[2, 5, 1], [33, 0, 70], [129, 64, 4]])
def test_many_tokens(new, dim, dtype):
    run([100, 0, 17], new, heads=2, groups=4, dim=dim, dtype=dtype)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 64, 100, 5000])
@pytest.mark.parametrize("new", [[1, 1], [7, 40]])
def test_windows(new, window):
    run([300, 20], new, window=window, groups=4, dtype="f16")


@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "bf16"), (256, "f16")])
def test_long(dim, dtype):
    """Several splits of many chunks, one request and a few."""
    run([9000], [1], heads=1, groups=5, dim=dim, page=128, dtype=dtype)
    run([3000, 5, 2000], [3, 1, 2], heads=1, groups=2, dim=dim, page=64, dtype=dtype)


@pytest.mark.parametrize("scaling", [0.0, -0.2, 1.0])
def test_scalings(scaling):
    """No scale weighs every token the same; a negative one turns the order; a large one leaves a single token."""
    run([77, 300], [1, 3], scaling=scaling, dtype="f32", spread=2.0)


def test_large_scores():
    run([500, 40], [1, 20], scaling=3.0, spread=30.0, dtype="f32")
    run([500, 40], [1, 20], scaling=3.0, spread=30.0, dtype="bf16")


def test_strided_queries_and_given_out():
    """Queries with heads before tokens in memory; rows behind the last request are left alone in a given out and are
    zeros in a new one."""
    cache, _ = build([50, 9], [1, 1], 2, 64, 16)
    step = cache.assign([2, 3], rows=9)
    cache.check()
    rows = torch.randn(9, 2, 64, device=DEV)
    cache.store(0, rows, rows, step)
    query = torch.randn(6, 9, 64, device=DEV).half().transpose(0, 1)
    out = torch.full((9, 6, 64), 7.0, dtype=torch.float16, device=DEV)
    assert cache.attend_rows(0, query, step, out=out) is out
    compare(cache, step, query, out, 64 ** -0.5)
    assert (out[5:] == 7.0).all()
    fresh = cache.attend_rows(0, query, step)
    assert torch.equal(fresh[:5], out[:5]) and not fresh[5:].any()
    odd = torch.randn(9, 6 * 64 + 3, device=DEV).half()[:, 3:].reshape(9, 6, 64)
    wide = torch.randn(9, 6, 65, device=DEV).half()[..., 1:]  # rows that are not 16-byte aligned are copied
    for q in (odd, wide):
        assert torch.equal(cache.attend_rows(0, q, step), cache.attend_rows(0, q.contiguous().clone(), step))


@pytest.mark.parametrize("longest,most", [(1, 1), (100000, 1000), (64, 3)])
def test_bounds_shape_launches_only(longest, most):
    """Bounds that are too small or too large leave the result what it is."""
    from paged_cache import Step

    cache, step = build([900, 2], [40, 3], 2, 64, 16)
    query = torch.randn(43, 4, 64, device=DEV).bfloat16()
    other = Step(step.slots, step.positions, step.cu, step.rows, longest, most)
    compare(cache, other, query, cache.attend_rows(0, query, other), 0.125)


def test_stale_pages_and_bad_table_entries():
    """What lies behind a request's tokens, NaN included, and table entries that are no page have no part."""
    cache, step = build([40, 21], [1, 1], 2, 128, 16)
    query = torch.randn(2, 6, 128, device=DEV).bfloat16()
    want = cache.attend_rows(0, query, step)
    held = torch.cat([cache.slots(0, 0, 41), cache.slots(1, 0, 22)])
    every = torch.arange(cache.pages * 16, device=DEV)
    rest = every[~torch.isin(every, held)]
    from paged_cache import Step

    bad = torch.full((len(rest), 2, 128), float("nan"), device=DEV)
    cache.store(0, bad, bad, Step(rest, rest, step.cu, len(rest), 1, 1))
    assert torch.equal(cache.attend_rows(0, query, step), want)
    # the second page of request 0 is gone: its other tokens are what is left
    keys, values = cache.load(0, cache.slots(0, 0, 41), torch.float32)
    keep = [t for t in range(41) if not 16 <= t < 32]
    for entry in (-1, cache.pages, 1 << 30):
        cache.table[0, 1] = entry
        got = cache.attend_rows(0, query, step)
        expect = paged_ref.attend(query[:1].double().cpu().numpy(), keys[keep].double().cpu().numpy(),
                                  values[keep].double().cpu().numpy(), 128 ** -0.5)
        assert np.abs(got[:1].double().cpu().numpy() - expect).max() <= (2 ** -8 + 2 ** -10) * values.abs().max().item()
        assert torch.equal(got[1], want[1])


def test_nan_reaches_only_rows_that_see_it():
    """A value block of NaN in the middle of a step's tokens: the tokens before it stay clean, those that see it get NaN
    in its dimensions; outside the window it is not seen."""
    cache, _ = build([30], [1], 1, 64, 16, room=2)
    step = cache.assign([20])
    cache.check()
    key, value = torch.randn(20, 1, 64, device=DEV), torch.randn(20, 1, 64, device=DEV)
    query = torch.randn(20, 2, 64, device=DEV)
    cache.store(0, key, value, step)
    clean = {w: cache.attend_rows(0, query, step, window=w) for w in (None, 4)}
    value[7, 0, 40] = float("nan")
    cache.store(0, key, value, step)
    for window, want in clean.items():
        got = cache.attend_rows(0, query, step, window=window)
        sees = torch.tensor([i >= 7 and (window is None or i < 7 + window) for i in range(20)], device=DEV)
        assert torch.equal(got[~sees], want[~sees])
        assert got[sees][..., 32:].isnan().all() and torch.equal(got[sees][..., :32], want[sees][..., :32])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("total,new", [(1, 1), (40, 3), (700, 1), (3000, 2), (200, 50)])
def test_nan_keys_and_queries(total, new, dtype):
    """A NaN query makes its own row NaN; a NaN key every row that sees it, also where a row sees nothing else, and in one
    split of many."""
    cache, step = build([total - new], [new], 1, 64, 16)
    query = torch.randn(new, 3, 64, device=DEV).to(TYPES[dtype])
    clean = cache.attend_rows(0, query, step)
    assert clean.isfinite().all()
    dirty = query.clone()
    dirty[-1, 1, 5] = float("nan")
    got = cache.attend_rows(0, dirty, step)
    assert got[-1, 1].isnan().all()
    got[-1, 1] = clean[-1, 1]
    assert torch.equal(got, clean)
    from paged_cache import Step

    slot = cache.slots(0, total - new, total - new + 1)  # the first of the new tokens
    key, value = cache.load(0, slot, torch.float32)
    key[0, 0, 3] = float("nan")
    cache.store(0, key, value, Step(slot, slot, step.cu, 1, 1, 1))
    assert cache.attend_rows(0, query, step).isnan().all()
    seen = cache.attend_rows(0, query, step, window=1)
    assert seen[0].isnan().all() and seen[1:].isfinite().all()


@pytest.mark.parametrize("total", [900, 1500, 20000])
def test_nan_value_of_no_weight(total):
    """A value of NaN that the softmax weighs by less than the smallest float32 makes its block NaN all the same, in one
    launch, joined in it or by another."""
    from paged_cache import Step

    cache, step = build([total - 1], [1], 1, 64, 16)
    query = torch.ones(1, 2, 64, device=DEV)
    key, value = torch.full((1, 1, 64), 6.0, device=DEV), torch.ones(1, 1, 64, device=DEV)
    value[0, 0, 33] = float("nan")
    for at, k in ((total - 1, key), (5, -key)):  # scores of 48 and -48, times 4: e^-384
        slot = cache.slots(0, at, at + 1)
        cache.store(0, k, value if at == 5 else torch.ones_like(value), Step(slot, slot, step.cu, 1, 1, 1))
    out = cache.attend_rows(0, query, step, scaling=0.5)
    assert out[..., 32:].isnan().all() and (out[..., :32] == 1.0).all()


def test_no_rows_and_no_tokens():
    cache, step = build([5, 0], [0, 0], 2, 64, 16)
    assert cache.attend_rows(0, torch.empty(0, 4, 64, device=DEV), step).shape == (0, 4, 64)
    # queries of requests that hold nothing (an assign that was refused): left as they are, or zeros
    step = cache.assign([10000, 1], rows=3)
    query = torch.randn(3, 4, 64, device=DEV)
    out = torch.full((3, 4, 64), 5.0, device=DEV)
    assert (cache.attend_rows(0, query, step, out=out) == 5.0).all()
    assert not cache.attend_rows(0, query, step).any()
    # more queries than tokens held: those before the first token see nothing
    cache.lengths.fill_(2)
    step.cu.copy_(torch.tensor([0, 3, 3], dtype=torch.int32))
    cache.table[0, 0] = 0
    got = cache.attend_rows(0, query, step)
    assert not got[0].any() and got[1:].isfinite().all()
    compare(cache, step, query, got, 0.125)


def test_layers_are_apart():
    cache, step = build([40], [2], 2, 64, 16, layers=3)
    query = torch.randn(2, 4, 64, device=DEV)
    compare(cache, step, query, cache.attend_rows(2, query, step), 0.125, layer=2)
    assert not cache.attend_rows(0, query, step).any()
    with pytest.raises(ValueError):
        cache.attend_rows(3, query, step)


def test_graph_and_streams():
    """Decode steps replayed from a graph, with eager work in between and another stream in use, equal eager ones."""
    cache, step = build([500, 90, 31], [1, 1, 1], 2, 128, 32, room=1)
    new = torch.ones(3, dtype=torch.int32, device=DEV)
    query, key, value = (torch.randn(3, h, 128, device=DEV) for h in (6, 2, 2))
    keep = cache.lengths.clone()

    def body():
        step = cache.assign(new, 3, longest=600, most=1)
        cache.store(0, key, value, step)
        return cache.attend_rows(0, query, step)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = body()
        cache.trim(keep)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body()
    for turn in range(4):
        graph.replay()
        cache.trim(keep)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and out.any(dim=-1).all(), turn
        out.fill_(float("nan"))
        want = body()
        cache.trim(keep)


@pytest.mark.parametrize("dim,lengths,new", [(64, [2900, 7], [1, 1]), (128, [700, 0, 40], [50, 3, 0]), (256, [1500], [20])])
def test_bounds_and_the_queries_place(dim, lengths, new):
    """Bounds that are too low, or far too high, change launches only; the result may take the queries' place."""
    cache, step = build(lengths, new, 2, dim, 16, seed=3)
    for longest in (1, max(lengths), 1 << 20):
        for most in (1, max(new), 4000):
            step.longest, step.most = longest, most
            query = torch.randn(step.rows, 8, dim, device=DEV).bfloat16()
            given = query.clone()
            got = cache.attend_rows(0, query, step, out=query)
            assert got.data_ptr() == query.data_ptr()
            compare(cache, step, given, got, dim ** -0.5)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_float16_weights_keep_their_low_bits(new, dim):
    """Values of 1 give 1 whatever the weights are.  Against the reference of the first 512 tokens the others weigh
    1 + 0.9 * 2^-11, which one float16 would round to 1: a mean of 1 - 0.8 * 2^-11, past half of the 2^-11 to the next
    float16 below 1.  Weights that are off by 2^-22 leave it next to 1."""
    from paged_cache import PagedCache

    total = 4096
    cache = PagedCache(1, 1, dim, total // 64 + 1, device=DEV)
    steps = cache.assign([total - new]), cache.assign([new])
    key = torch.zeros(total, 1, dim, device=DEV)
    key[512:, 0, 0] = 1.0
    value = torch.ones(total, 1, dim, device=DEV)
    for step, rows in zip(steps, (slice(0, total - new), slice(total - new, total))):
        cache.store(0, key[rows], value[rows], step)
    steps[1].longest = 1  # no splits: one reference for all tokens
    query = torch.zeros(new, 2, dim, device=DEV, dtype=torch.float16)
    query[..., 0] = 1.0
    out = cache.attend_rows(0, query, steps[1], scaling=float(np.log1p(0.9 * 2.0 ** -11)))
    assert torch.equal(out, torch.ones_like(out))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,total,new,window", [(1, 1, 1, None), (1, 700, 1, None), (1, 3000, 2, None), (1, 20000, 1, None),
                                                    (1, 200, 50, None), (1, 200, 50, 20), (1, 6000, 300, None), (8, 5000, 700, None)])
def test_scores_of_minus_infinity(heads, total, new, window, dtype):
    """A row that sees tokens, all with scores of -infinity, is NaN (0 / 0), unlike one that sees none; other rows keep
    their results, in one launch, joined in it or by the others."""
    cache, step = build([total - new], [new], heads, 64, 64)
    from paged_cache import Step

    slots = cache.slots(0, 0, total)
    key, value = cache.load(0, slots, torch.float32)
    key[..., 0] = 1.0  # (a key of 0 would make NaN of itself)
    cache.store(0, key, value, Step(slots, slots, step.cu, total, 1, 1))
    assert (cache.load(0, slots, torch.float32)[0][..., 0] > 0).all()
    query = torch.randn(new, 3 * heads, 64, device=DEV).to(TYPES[dtype])
    clean = cache.attend_rows(0, query, step, window=window)
    assert clean.isfinite().all()
    rows = sorted({0, new // 2, new - 1})
    query[rows, 1, 0] = -float("inf")
    got = cache.attend_rows(0, query, step, window=window)
    assert got[rows, 1].isnan().all()
    got[rows, 1] = clean[rows, 1]
    assert torch.equal(got, clean)
    cache.table.fill_(-1)  # no page holds a token: nothing is seen
    assert not cache.attend_rows(0, query, step, window=window).any()


def test_results_over_other_queries_are_refused():
    cache, step = build([50, 9], [2, 3], 2, 64, 16)
    room = torch.randn(8, 6, 64, device=DEV)
    given = room.clone()
    want = cache.attend_rows(0, given[:5], step)
    for out in (room[1:6], room.view(-1)[64:64 + 5 * 384].view(5, 6, 64)):
        with pytest.raises(ValueError, match="other rows"):
            cache.attend_rows(0, room[:5], step, out=out)
    assert torch.equal(room, given)
    assert torch.equal(cache.attend_rows(0, room[:5], step, out=room[:5]), want)


@pytest.mark.parametrize("given", ["nothing", "a result", "the query's place"])
def test_recorded_calls_have_no_gradient(given):
    """Attention has no backward pass: a recorded call's result is the plain one, requires a gradient and refuses it."""
    cache, step = build([50, 9], [2, 3], 2, 64, 16)
    query = torch.randn(5, 6, 64, device=DEV)
    want = cache.attend_rows(0, query, step)
    assert not want.requires_grad
    leaf = query.clone().requires_grad_()
    rows = leaf * 1.0
    out = {"nothing": None, "a result": torch.empty_like(query), "the query's place": rows}[given]
    got = cache.attend_rows(0, rows, step, out=out)
    assert got.requires_grad and torch.equal(got, want) and (out is None or got is out)
    with pytest.raises(RuntimeError, match="no backward pass"):
        got.sum().backward()
    with torch.no_grad():
        assert not cache.attend_rows(0, leaf, step).requires_grad


def test_a_recorded_leaf_is_not_written():
    """What autograd does not let change in place stays as it is."""
    cache, step = build([50, 9], [2, 3], 2, 64, 16)
    leaf = torch.randn(5, 6, 64, device=DEV).requires_grad_()
    given = leaf.detach().clone()
    for place in (leaf, leaf[:]):
        with pytest.raises(RuntimeError, match="leaf"):
            cache.attend_rows(0, leaf, step, out=place)
    assert torch.equal(leaf, given)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("total,new", [(40, 1), (600, 1), (64, 64), (3000, 20)])
def test_scores_of_the_last_products(total, new, dim, dtype):
    """Scores that are large in the last matrix instruction of a tile alone, one tile after the other: read before that has
    ended they would be 0, and the weights, against a reference of 0, infinite.  All tokens but one score 0 and that one
    e^60 times their weight, so the result is its value, but for total values of 6 at the most that weigh e^-60 each."""
    from paged_cache import PagedCache

    cache = PagedCache(1, 1, dim, -(-total // 64) + 1, device=DEV)
    cache.assign([total - new])
    step = cache.assign([new])
    slots = cache.slots(0, 0, total)
    from paged_cache import Step

    steps = dim // 32
    dims = [g * (dim // 4) + (steps - 1) * 8 + j for g in range(4) for j in range(8)]  # the last step's
    value = torch.arange(total, device=DEV).remainder(6).float()[:, None, None].expand(total, 1, dim).contiguous()
    query = torch.zeros(new, 2, dim, device=DEV, dtype=TYPES[dtype])
    query[..., dims] = 1.0
    for at in {0, 3, 17, total // 2, total - new}:
        key = torch.zeros(total, 1, dim, device=DEV)
        key[at, 0, dims] = 6.0
        cache.store(0, key, value, Step(slots, slots, step.cu, total, 1, 1))
        held = cache.load(0, slots[at:at + 1], torch.float32)[1][0, 0, 0].item()
        out = cache.attend_rows(0, query, step, scaling=60.0 / (6.0 * len(dims)))
        seen = step.positions >= at
        assert (out[seen].float() - held).abs().max() <= 2.0 ** -8 * held + 6 * total * np.exp(-60.0), (at, out[seen].float().max())
