"""Attention of shaped scores over the paged 4-bit cache against the formula in 64 bits on the values the cache holds
(oracle/paged_ref.attend_shaped, which test_formula_of_compare holds compare to).

A result may be off by its type's rounding u |ref| and by what the errors of its weights weigh.  Token t's weight p_t is off
by the relative error of its exponential, d_t = w + s_t: w for the pieces a weight is held in (2^-11, in two pieces 2^-22),
s_t the error of its score.  So the sum is off by sum p_t d_t |v_t|, and what it is divided by, relative to it, by
sum p_t d_t and the sums' own n 2^-24.  s_t in units of 2^-24: D + 8 roundings of the products on sum |q k| scaling, two of
the exponent's argument and two units of the exponential (2 |z| + 32), three of the bias and its sum (3 |bias|), and a
capped score's: cap tanh(u) of a float32 u is 8 |z| off at the most where it is a polynomial times u, and where it is
cap - 2 cap / (1 + e^2u) the parts of that are cap in size: 12 cap, taken only if a score reaches half of the cap, so
12 min(cap, 2 max |z|).  Bfloat16 results take the second form under every cap up to 128, whose 12 * 128 * 2^-24 is less than
the 2^-12 that w has above half a step of a float16.  The smallest weights are subnormal float16, as in test_gpu_paged_attend.  A float16 result below
2^-14 is subnormal too: its steps are 2^-24 whatever its size, so its rounding is off by 2^-25 and not by 2^-11 |ref|."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_ref
from test_gpu_paged_attend import DEV, STEP, TYPES, build

pytestmark = pytest.mark.gpu
PIECES = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -11}


def formula(q, k, v, scaling, position, low, high, cap, slope, sink):
    """(result, bound without the type's rounding) of one row over keys and values [total, D]."""
    at = np.arange(low, high + 1)
    k, v = k[at], v[at]
    z = k @ q * scaling
    unit = (k.shape[1] + 8) * (np.abs(k) @ np.abs(q)) * abs(scaling) + 40
    if cap is not None:
        unit = unit + 8 * np.abs(z) + 12 * min(cap, 2 * np.abs(z).max())
        z = cap * np.tanh(z / cap)
    bias = slope * np.abs(position - at)
    z = z - bias
    unit = unit + 2 * np.abs(z) + 3 * np.abs(bias)
    top = max(z.max(), sink)
    p = np.exp(z - top)
    p /= p.sum() + np.exp(sink - top)
    return p @ v, p, unit, v


def compare(cache, step, query, got, scaling=None, window=None, cap=None, slopes=None, sinks=None, first=None, last=None,
            layer=0, heads=None, some=None):
    """Every row and head (or the query heads, and the rows of a request, given) against the formula, with the bound above."""
    lengths, cu, dtype, dim = cache.lengths.tolist(), step.cu.tolist(), query.dtype, cache.head_dim
    scaling = dim ** -0.5 if scaling is None else scaling
    slopes, sinks, first, last = (None if t is None else t.double().cpu().numpy() if t.is_floating_point() else t.tolist()
                                  for t in (slopes, sinks, first, last))
    groups = query.shape[1] // cache.kv_heads
    for b, total in enumerate(lengths):
        lo, hi = cu[b], cu[b + 1]
        if lo == hi:
            continue
        keys, values = (t.double().cpu().numpy() for t in cache.load(layer, cache.slots(b, 0, total), torch.float32))
        q, have = (t[lo:hi].double().cpu().numpy() for t in (query, got))
        for i in range(hi - lo) if some is None else sorted({min(x, hi - lo - 1) for x in some}):
            position = total - (hi - lo) + i
            low = 0 if first is None else max(first[lo + i], 0)
            low = low if window is None else max(low, position - window + 1)
            high = min(position if last is None else last[lo + i], total - 1)
            for h in range(q.shape[1]) if heads is None else heads:
                if high < low:
                    assert not have[i, h].any(), (b, i, h)
                    continue
                want, p, unit, v = formula(q[i, h], keys[:, h // groups], values[:, h // groups], scaling, position, low, high, cap,
                                           0.0 if slopes is None else slopes[h], -np.inf if sinks is None else sinks[h])
                d = PIECES[dtype] + 2.0 ** -24 * unit
                size = p @ np.abs(v)
                bound = STEP[dtype] * np.abs(want) + (2.0 ** -25 if dtype == torch.float16 else 0.0) + (p * d) @ np.abs(v) + ((p * d).sum() + (len(p) + 8) * 2.0 ** -24) * size
                bound += (2.0 ** -40 if dtype == torch.float32 else 2.0 ** -33) * np.abs(v).sum(0)
                error = np.abs(have[i, h] - want)
                assert (error <= bound).all(), (b, i, h, error.max(), (error / np.maximum(bound, 1e-300)).max())


def numbers(n, seed, scale=1.0):
    return (torch.randn(n, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV)


def shape_of(kind, rows, heads, step, lengths):
    """Arguments of a kind of shape: its words joined by +."""
    made = {}
    for word in kind.split("+"):
        if word.startswith("cap"):
            made["cap"] = float(word[3:])
        elif word == "slopes":
            made["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device=DEV).float() / heads)
        elif word == "sinks":
            made["sinks"] = numbers(heads, 5, 2.0)
        elif word.startswith("window"):
            made["window"] = int(word[6:])
        elif word == "documents":
            g = torch.Generator().manual_seed(rows)
            made["first"] = (torch.rand(rows, generator=g).to(DEV) * (step.positions + 2)).long()  # past a row's own, some
        elif word.startswith("prefix"):
            made["last"] = torch.maximum(step.positions, torch.full_like(step.positions, int(word[6:]) - 1))
    return made


def run(kind, lengths, new, heads=2, groups=3, dim=64, page=16, dtype="bf16", seed=0, reach=3.0, only=None, some=None, scaling=None):
    print(f"[case] shaped {kind} {lengths} + {new} heads={heads}x{groups} dim={dim} page={page} {dtype}", flush=True)
    cache, step = build(lengths, new, heads, dim, page, seed)
    g = torch.Generator(DEV).manual_seed(seed + 1)
    query = (torch.randn(step.rows, heads * groups, dim, generator=g, device=DEV) * reach).to(TYPES[dtype])
    made = shape_of(kind, step.rows, heads * groups, step, lengths)
    got = cache.attend_rows(0, query, step, scaling=scaling, **made)
    assert got.shape == query.shape and got.dtype == query.dtype
    compare(cache, step, query, got, scaling=scaling, heads=only, some=some, **made)
    return cache, step, query, made, got


KINDS = ["cap5", "slopes", "sinks", "documents", "prefix30", "cap20+slopes+sinks+documents+window50"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,page,dtype", [(64, 16, "f32"), (64, 32, "bf16"), (128, 64, "f16"), (128, 16, "bf16"), (256, 32, "bf16"),
                                            (256, 64, "f32")])
def test_single_tokens(kind, dim, page, dtype):
    """Lengths of one token, around a tile, a chunk, a page and a split."""
    run(kind, [0, 1, 14, 15, 16, 47, 62, 63, 64, 65, 200, 255, 256, 700], [1] * 14, dim=dim, page=page, dtype=dtype)


@pytest.mark.parametrize("kind", KINDS + ["cap8+prefix70", "slopes+prefix41+sinks"])
@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (64, "f32"), (128, "bf16"), (128, "f32"), (256, "bf16"), (256, "f32")])
def test_many_tokens(kind, dim, dtype):
    run(kind, [100, 0, 17], [33, 0, 70], groups=4, dim=dim, dtype=dtype)
    run(kind, [40, 3], [2, 5], groups=2, dim=dim, dtype=dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,groups", [(1, 1), (3, 1), (8, 4), (2, 7), (1, 16), (1, 20), (2, 40)])
def test_heads(heads, groups, dtype):
    """A slope and a sink of its own for each query head."""
    run("cap6+slopes+sinks", [130, 3], [1, 1], heads=heads, groups=groups, dim=128, page=32, dtype=dtype)


@pytest.mark.parametrize("kind", ["cap10+sinks", "slopes+sinks", "documents+sinks", "window700+sinks+cap15"])
@pytest.mark.parametrize("dim,dtype", [(64, "f32"), (128, "bf16"), (256, "f16")])
def test_long(kind, dim, dtype):
    """Several splits of many chunks, joined in the launch and by others; one request and a few."""
    run(kind, [9000], [1], heads=1, groups=5, dim=dim, page=128, dtype=dtype)
    run(kind, [20000], [2], heads=2, groups=2, dim=dim, page=64, dtype=dtype)
    run(kind, [3000, 5, 2000], [3, 1, 2], heads=1, groups=2, dim=dim, page=64, dtype=dtype)
    run(kind, [5000], [200], heads=8, groups=4, dim=dim, page=64, dtype=dtype, only=[0, 13, 31])


@pytest.mark.parametrize("kind,heads,new", [("documents+sinks", 8, [2200]), ("documents+cap6+slopes", 8, [2100, 0, 300]),
                                            ("cap9+window500", 8, [4200]), ("slopes+window64+sinks", 8, [4100, 40]),
                                            ("cap12+sinks", 16, [8210]), ("slopes+prefix700", 16, [8210]), ("documents", 16, [8210])])
@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16"), (64, "bf16"), (128, "f16")])
def test_many_blocks(kind, heads, new, dim, dtype):
    """Prompts of so many blocks of 64 rows that two waves, or one, take each: rows around blocks, tiles and the ends."""
    run(kind, [0] * len(new), new, heads=heads, groups=4, dim=dim, page=64, dtype=dtype, only=[0, 5, 4 * heads - 1],
        some=[0, 1, 15, 16, 17, 39, 500, 699, 700, 701, 1039, 2079, 2199, new[0] // 2, new[0] - 17, new[0] - 1])


@pytest.mark.parametrize("heads,kind,dim,dtype", [(2, "window100+cap5+sinks", 64, "bf16"), (1, "documents+window90", 64, "f16"),
                                                  (2, "slopes+window70", 128, "bf16")])
def test_more_blocks_than_a_launch(heads, kind, dim, dtype):
    """Prompts of more than 4,096 blocks of rows: a workgroup takes several, one after the other."""
    new = 40000
    run(kind, [0], [new], heads=heads, groups=8, dim=dim, page=64, dtype=dtype, only=[0, 8 * heads - 1],
        some=[0, 1, 17, 99, 100, 3615, 7232, 7233, 8191, 8192, 20000, 32767, 32768, new - 2, new - 1])


def test_pages_past_32_bits():
    """Rows appended to, and attended to in, pages whose codes lie past 2^32 bytes."""
    from paged_cache import PagedCache, Step
    from test_gpu_paged_append import check, inputs, tables

    page, heads, dim = 64, 8, 256
    pages = (1 << 32) // (heads * page * dim // 2) + 5
    cache = PagedCache(1, heads, dim, pages, page=page, requests=1, table_pages=2, device=DEV)
    cache.table.copy_(torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32))
    cache.lengths.fill_(100)
    slots = cache.slots(0, 0, 100)
    assert int(slots.min()) * heads * dim // 2 > 1 << 32
    step = Step(slots, torch.arange(100, device=DEV), torch.tensor([0, 100], dtype=torch.int32, device=DEV), 100, 100, 100)
    query, key, value = inputs(100, 16, heads, dim, "bf16")
    cos, sin = tables(100, dim // 2)
    turned = cache.append(0, query, key, value, step, cos, sin)
    check(cache, step, query, key, value, turned, cos, sin)
    made = dict(cap=6.0, sinks=numbers(16, 2))
    compare(cache, step, turned, cache.attend_rows(0, turned, step, **made), heads=[0, 15], some=[0, 50, 99], **made)


@pytest.mark.parametrize("kind", ["documents+sinks", "window300+cap7"])
def test_many_blocks_against_few(kind):
    """Every row of a launch of one or two waves a block against the same rows in a launch of four, to what two roundings of
    the results and the orders of sums may differ (twice 2^-8, and 2^-9 for weights of one float16)."""
    cache, step = build([0], [4200], 8, 64, 64)
    query = torch.randn(step.rows, 32, 64, generator=torch.Generator(DEV).manual_seed(5), device=DEV).bfloat16()
    made = shape_of(kind, step.rows, 32, step, [0])
    want = cache.attend_rows(0, query, step, **made)
    from paged_cache import Step

    other = Step(step.slots, step.positions, step.cu, step.rows, step.longest, 100)  # a bound on rows that shapes fewer blocks
    got = cache.attend_rows(0, query, other, **made)
    assert torch.equal(want.any(-1), got.any(-1))  # rows that see nothing
    size = cache.load(0, step.slots, torch.float32)[1].abs().max().item()
    assert (got.float() - want.float()).abs().max().item() <= (2.0 ** -7 + 2.0 ** -9) * size


@pytest.mark.parametrize("cap", [1e-3, 0.4, 3.0, 1e4, 1e9])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_caps(cap, dtype):
    """From a cap that all scores reach to one that none comes near; scores of all sizes beside each other."""
    run(f"cap{cap}", [77, 300], [1, 40], dtype=dtype, reach=1.0)
    cache, step = build([290], [10], 1, 64, 16)
    query = torch.randn(10, 3, 64, device=DEV).to(TYPES[dtype])
    query[3:6] *= 60.0
    query[6:8] *= 1e-4
    compare(cache, step, query, cache.attend_rows(0, query, step, cap=cap), cap=cap)


@pytest.mark.parametrize("scaling", [0.0, -0.2, 2.0])
def test_scalings(scaling):
    """Scores turned round by a negative scale; the distance's bias is not."""
    run("cap4+slopes", [77, 300], [1, 3], scaling=scaling, dtype="f32")
    run("slopes+sinks", [77, 300], [1, 30], scaling=scaling, dtype="bf16")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_a_scale_that_is_no_number(dtype):
    cache, step = build([77, 300], [1, 30], 1, 64, 16)
    query = torch.randn(31, 2, 64, device=DEV).to(TYPES[dtype])
    for made in (dict(cap=5.0), dict(cap=5.0, slopes=numbers(2, 1)), dict(slopes=numbers(2, 1)), dict(sinks=numbers(2, 1))):
        assert cache.attend_rows(0, query, step, scaling=float("nan"), **made).isnan().all()


@pytest.mark.parametrize("new", [1, 45])
def test_slopes_and_sinks_of_any_size(new):
    cache, step = build([400], [new], 1, 64, 16)
    query = torch.randn(new, 8, 64, device=DEV)
    slopes = torch.tensor([0.0, -0.01, 5.0, 1e-6, 0.5, 0.1, -0.3, 100.0], device=DEV)
    compare(cache, step, query, cache.attend_rows(0, query, step, slopes=slopes), slopes=slopes)
    sinks = torch.tensor([-float("inf"), -80.0, 0.0, 3.0, 30.0, 100.0, 1e4, 1.0], device=DEV)
    got = cache.attend_rows(0, query, step, sinks=sinks)
    compare(cache, step, query, got, sinks=sinks)
    assert not got[:, 6].any()  # e^-10000
    bare = cache.attend_rows(0, query, step, first=torch.zeros(new, dtype=torch.int64, device=DEV))
    assert torch.equal(got[:, 0], bare[:, 0])


@pytest.mark.parametrize("total,new", [(60, 60), (700, 1), (9000, 3)])
def test_ranges_that_leave_nothing(total, new):
    """Rows whose range is empty, before the first token, behind the last or turned round are 0, with sinks too; neighbours
    keep their results.  Ends far outside of 32 bits are ends all the same."""
    far = 1 << 62
    cache, step = build([total - new], [new], 2, 64, 16)
    query = torch.randn(new, 6, 64, device=DEV).bfloat16()
    sinks = numbers(6, 3)
    for first, last in ((total, total + 5), (-far, -1), (30, 29), (far, -far), (far, far), (0, -far)):
        low, high = step.positions * 0, step.positions.clone()
        low[-1], high[-1] = first, last
        got = cache.attend_rows(0, query, step, sinks=sinks, first=low, last=high)
        assert not got[-1].any()
        compare(cache, step, query, got, sinks=sinks, first=low, last=high)
    whole = cache.attend_rows(0, query, step, first=torch.full_like(step.positions, -far), last=torch.full_like(step.positions, far))
    compare(cache, step, query, whole, last=step.positions * 0 + total)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_infinite_scores_reach_the_cap(dtype):
    """Queries of infinity where no key is 0: scores of the cap, up or down; without a cap the row is NaN."""
    from paged_cache import Step

    cache, step = build([60], [40], 1, 64, 16)
    slots = cache.slots(0, 0, 100)
    key, value = cache.load(0, slots, torch.float32)
    key[..., 7] = torch.where(torch.arange(100, device=DEV) % 3 == 0, 4.0, -4.0)[:, None]
    key[..., :7] = key[..., 8:32] = 4.0
    cache.store(0, key, value, Step(slots, slots, step.cu, 100, 1, 1))
    query = torch.zeros(40, 2, 64, device=DEV)
    query[:, 0, 7] = 1e30 if dtype != "f16" else 6e4
    query[:, 1, 7] = -1e30 if dtype != "f16" else -6e4
    query = query.to(TYPES[dtype])
    finite = cache.attend_rows(0, query, step, cap=3.0)
    compare(cache, step, query, finite, cap=3.0)
    endless = query.float()
    endless[..., 7] *= float("inf")
    endless[..., :7] = endless[..., 8:] = 0.0
    endless = torch.nan_to_num(endless, nan=0.0, posinf=float("inf"), neginf=-float("inf")).to(TYPES[dtype])
    got = cache.attend_rows(0, endless, step, cap=3.0)
    assert torch.equal(got, finite)
    assert cache.attend_rows(0, endless, step, sinks=numbers(2, 1)).isnan().all()


def test_stale_pages_and_bad_table_entries():
    """What lies outside of a row's tokens, NaN included, and table entries that are no page have no part."""
    from paged_cache import Step

    cache, step = build([40, 21], [1, 1], 2, 128, 16)
    query = torch.randn(2, 6, 128, device=DEV).bfloat16()
    made = dict(cap=4.0, slopes=numbers(6, 2).abs(), sinks=numbers(6, 3))
    last = torch.full((2,), 1 << 40, dtype=torch.int64, device=DEV)  # as far as the request goes
    want = cache.attend_rows(0, query, step, last=last, **made)
    held = torch.cat([cache.slots(0, 0, 41), cache.slots(1, 0, 22)])
    every = torch.arange(cache.pages * 16, device=DEV)
    rest = every[~torch.isin(every, held)]
    bad = torch.full((len(rest), 2, 128), float("nan"), device=DEV)
    cache.store(0, bad, bad, Step(rest, rest, step.cu, len(rest), 1, 1))
    assert torch.equal(cache.attend_rows(0, query, step, last=last, **made), want)
    for entry in (-1, cache.pages, 1 << 30):
        cache.table[0, 1] = entry
        got = cache.attend_rows(0, query, step, **made)
        assert got.isfinite().all() and torch.equal(got[1], want[1]) and not torch.equal(got[0], want[0])


@pytest.mark.parametrize("total,new", [(40, 20), (3000, 30), (3000, 2)])
def test_nan_reaches_only_rows_that_see_it(total, new):
    """A value of NaN makes its block NaN in the rows whose range holds the token, a key of NaN the whole row; the others
    keep their bits."""
    from paged_cache import Step

    cache, step = build([total - new], [new], 1, 64, 16)
    query = torch.randn(new, 2, 64, device=DEV)
    first = (step.positions - 6).clamp(min=0)
    first[::2] = 0
    made = dict(first=first, slopes=torch.full((2,), 0.01, device=DEV), cap=9.0, sinks=numbers(2, 4))
    clean = cache.attend_rows(0, query, step, **made)
    at = total - new // 2 - 1
    slot = cache.slots(0, at, at + 1)
    key, value = cache.load(0, slot, torch.float32)
    sees = (first <= at) & (step.positions >= at)
    assert sees.any()
    dirty = value.clone()
    dirty[0, 0, 40] = float("nan")
    cache.store(0, key, dirty, Step(slot, slot, step.cu, 1, 1, 1))
    got = cache.attend_rows(0, query, step, **made)
    assert torch.equal(got[~sees], clean[~sees])
    assert got[sees][..., 32:].isnan().all() and torch.equal(got[sees][..., :32], clean[sees][..., :32])
    key[0, 0, 3] = float("nan")
    cache.store(0, key, value, Step(slot, slot, step.cu, 1, 1, 1))
    got = cache.attend_rows(0, query, step, **made)
    assert torch.equal(got[~sees], clean[~sees]) and got[sees].isnan().all()


def test_padded_rows_strides_and_places():
    """Rows behind the last request are left alone in a given out and zeros in a new one; strided queries; the result in the
    queries' place."""
    cache, _ = build([50, 9], [1, 1], 2, 64, 16)
    step = cache.assign([2, 3], rows=9)
    cache.check()
    rows = torch.randn(9, 2, 64, device=DEV)
    cache.store(0, rows, rows, step)
    query = torch.randn(6, 9, 64, device=DEV).half().transpose(0, 1)
    made = dict(cap=3.0, slopes=numbers(6, 1).abs(), sinks=numbers(6, 2), first=torch.zeros(9, dtype=torch.int64, device=DEV),
                last=step.positions.clone())
    out = torch.full((9, 6, 64), 7.0, dtype=torch.float16, device=DEV)
    assert cache.attend_rows(0, query, step, out=out, **made) is out
    compare(cache, step, query, out, **made)
    assert (out[5:] == 7.0).all()
    fresh = cache.attend_rows(0, query, step, **made)
    assert torch.equal(fresh[:5], out[:5]) and not fresh[5:].any()
    wide = torch.randn(9, 6, 65, device=DEV).half()[..., 1:]  # rows that are not 16-byte aligned are copied
    want = cache.attend_rows(0, wide, step, **made)
    held = wide.contiguous()
    assert torch.equal(cache.attend_rows(0, held, step, out=held, **made)[:5], want[:5])
    room = torch.randn(10, 6, 64, device=DEV)
    with pytest.raises(ValueError, match="other rows"):
        cache.attend_rows(0, room[:9], step, out=room[1:], cap=2.0)


def test_refusals():
    cache, step = build([50], [3], 2, 64, 16)
    query = torch.randn(3, 4, 64, device=DEV)
    for bad in (dict(cap=0.0), dict(cap=-2.0), dict(cap=float("inf")), dict(slopes=torch.zeros(3, device=DEV)),
                dict(slopes=torch.zeros(4)), dict(sinks=torch.zeros(4, device=DEV).half()), dict(sinks=torch.zeros(8, device=DEV)[::2]),
                dict(first=torch.zeros(2, dtype=torch.int64, device=DEV)), dict(last=torch.zeros(3, dtype=torch.int32, device=DEV)),
                dict(window=0, cap=2.0)):
        with pytest.raises(ValueError):
            cache.attend_rows(0, query, step, **bad)
    none = torch.empty(0, 4, 64, device=DEV)
    empty = cache.assign([0])
    assert cache.attend_rows(0, none, empty, cap=3.0, first=empty.positions).shape == (0, 4, 64)


@pytest.mark.parametrize("longest,most", [(1, 1), (100000, 1000), (64, 3)])
def test_bounds_shape_launches_only(longest, most):
    from paged_cache import Step

    cache, step = build([900, 2], [40, 3], 2, 64, 16)
    query = torch.randn(43, 4, 64, device=DEV).bfloat16()
    other = Step(step.slots, step.positions, step.cu, step.rows, longest, most)
    made = dict(cap=5.0, sinks=numbers(4, 1), slopes=numbers(4, 2).abs(), first=(step.positions - 300).clamp(min=0))
    compare(cache, other, query, cache.attend_rows(0, query, other, **made), **made)


def test_more_queries_than_tokens():
    """Rows before the first token see nothing of their own accord, and what a given last lets them see."""
    cache, step = build([5, 0], [0, 0], 2, 64, 16)
    step = cache.assign([0, 0], rows=3)
    query = torch.randn(3, 4, 64, device=DEV)
    cache.lengths.fill_(2)
    step.cu.copy_(torch.tensor([0, 3, 3], dtype=torch.int32))
    got = cache.attend_rows(0, query, step, cap=2.0)
    assert not got[0].any() and got[1:].any()
    compare(cache, step, query, got, cap=2.0)
    last = torch.full((3,), 1, dtype=torch.int64, device=DEV)
    slopes = numbers(4, 1).abs()
    compare(cache, step, query, cache.attend_rows(0, query, step, last=last, slopes=slopes), last=last, slopes=slopes)


def test_distances_past_24_bits():
    """Two tokens far apart in a request of 2^25 tokens: the nearer distances stay whole numbers."""
    from paged_cache import PagedCache

    total, page = (1 << 25) + 37, 4096
    cache = PagedCache(1, 1, 64, 3, page=page, requests=1, table_pages=-(-total // page) + 1, device=DEV)
    last_page = (total - 1) // page
    cache.table.fill_(-1)
    cache.table[0, 0], cache.table[0, last_page] = 0, 1
    cache.lengths.fill_(total)
    g = torch.Generator(DEV).manual_seed(2)
    rows = torch.randn(2 * page, 1, 64, generator=g, device=DEV)
    from paged_cache import Step
    slots = torch.arange(2 * page, device=DEV)
    cu = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    cache.store(0, rows, rows.flip(0).contiguous(), Step(slots, slots, cu, 2 * page, 1, 1))
    query = torch.randn(2, 2, 64, generator=g, device=DEV)
    step = Step(slots[:2], torch.tensor([total - 2, total - 1], device=DEV), cu, 2, total, 2)
    slopes = torch.tensor([0.25, 3e-8], device=DEV)
    got = cache.attend_rows(0, query, step, slopes=slopes)
    keys, values = (t.double().cpu().numpy() for t in cache.load(0, slots, torch.float32))
    place = np.concatenate([np.arange(page), last_page * page + np.arange(page)])
    for i in range(2):
        position = total - 2 + i
        sees = place <= position
        for h in range(2):
            z = keys[sees, 0] @ query[i, h].double().cpu().numpy() * 0.125 - float(slopes[h]) * (position - place[sees])
            p = np.exp(z - z.max())
            want = (p / p.sum()) @ values[sees, 0]
            assert np.abs(got[i, h].double().cpu().numpy() - want).max() < 2e-5


def test_graph_streams_and_changed_tensors():
    """Two captured steps on one cache, replayed in turn with eager work and another stream between: each replay reads the
    shapes' tensors as they are then."""
    cache, step = build([5000, 90, 31], [1, 1, 1], 2, 128, 32, room=1)
    new = torch.ones(3, dtype=torch.int32, device=DEV)
    query, key, value = (torch.randn(3, h, 128, device=DEV) for h in (6, 2, 2))
    keep = cache.lengths.clone()
    slopes, sinks, first = numbers(6, 1).abs(), numbers(6, 2), torch.zeros(3, dtype=torch.int64, device=DEV)

    def body(**made):
        step = cache.assign(new, 3, longest=6000, most=1)
        cache.store(0, key, value, step)
        return cache.attend_rows(0, query, step, **made)

    shapes = [dict(cap=7.0, sinks=sinks), dict(slopes=slopes, first=first)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for made in shapes:
            body(**made)
            cache.trim(keep)
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for made in shapes:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = body(**made)
        graphs.append((graph, out, made))
    for turn in range(4):
        sinks.add_(0.5)
        first.add_(3)
        for graph, out, made in graphs:
            graph.replay()
            cache.trim(keep)
            torch.cuda.synchronize()
            want = body(**made)
            cache.trim(keep)
            assert torch.equal(out, want) and out.any(dim=-1).all(), turn
            out.fill_(float("nan"))


@pytest.mark.parametrize("of", ["query", "sinks", "slopes"])
def test_recorded_calls_have_no_gradient(of):
    cache, step = build([50, 9], [2, 3], 2, 64, 16)
    given = dict(query=torch.randn(5, 6, 64, device=DEV), sinks=numbers(6, 1), slopes=numbers(6, 2).abs())
    want = cache.attend_rows(0, given["query"], step, sinks=given["sinks"], slopes=given["slopes"])
    assert not want.requires_grad
    given[of].requires_grad_()
    got = cache.attend_rows(0, given["query"], step, sinks=given["sinks"], slopes=given["slopes"])
    assert got.requires_grad and torch.equal(got, want)
    with pytest.raises(RuntimeError, match="no backward pass"):
        got.sum().backward()


def test_formula_of_compare():
    """The comparison's formula is the oracle's."""
    rng = np.random.RandomState(4)
    query, keys, values = rng.randn(3, 2, 64), rng.randn(9, 1, 64), rng.randn(9, 1, 64)
    slopes, sinks, first, last = rng.rand(2), rng.randn(2), [0, 3, 2], [4, 8, 30]
    want = paged_ref.attend_shaped(query, keys, values, 0.2, 7, 1.5, slopes, sinks, first, last)
    for i in range(3):
        low, high = max(first[i], 6 + i - 6), min(last[i], 8)
        for h in range(2):
            assert np.allclose(formula(query[i, h], keys[:, 0], values[:, 0], 0.2, 6 + i, low, high, 1.5, slopes[h], sinks[h])[0], want[i, h])
