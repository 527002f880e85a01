"""The paged 4-bit cache on the GPU against oracle/paged_ref.py: tables and slots exactly, stored values exactly (a
value of the cache is a float16, bfloat16 and float32 value), over page sizes, types, strides, slots that run over page
ends, rows without a slot, blocks with infinities and NaN, the smallest and largest magnitudes."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def int32(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEV)


def make(requests=3, width=6, pages=16, page=16, layers=1, heads=2, dim=64):
    from paged_cache import PagedCache

    cache = PagedCache(layers, heads, dim, pages, page=page, requests=requests, table_pages=width, device=DEV)
    return cache, paged_ref.Tables(requests, width, pages, page)


def check_tables(cache, ref):
    assert cache.lengths.tolist() == ref.lengths
    assert int(cache.free_count) == len(ref.free)
    assert cache.free[:len(ref.free)].tolist() == ref.free
    for row, want in zip(cache.table.tolist(), ref.table):
        assert row == want + [-1] * (cache.table_pages - len(want))


def check_step(step, want):
    slots, positions, cu, _ = want
    assert step.slots.tolist() == slots
    assert step.positions.tolist() == positions
    assert step.cu.tolist() == cu


@pytest.mark.parametrize("requests,page", [(1, 16), (3, 32), (64, 16), (65, 64), (1025, 16), (2500, 128), (8192, 16)])
def test_assign_and_trim(requests, page):
    """Admissions, single tokens, ends and cuts in any order, the tables equal after each."""
    rng = np.random.RandomState(requests)
    width = 5
    cache, ref = make(requests, width, requests * 3 + 2, page, heads=1)
    for turn in range(8):
        print(f"[case] assign requests={requests} page={page} turn={turn}", flush=True)
        room = width * page - np.array(ref.lengths)
        kind = turn % 4
        new = np.minimum(room, 1 if kind == 1 else rng.randint(0, 2 * page, requests))
        if kind == 3:
            new[rng.randint(0, requests)] = -4  # taken as none
        rows = int(np.maximum(new, 0).sum()) + int(rng.choice([0, 3]))
        step = cache.assign(int32(new), rows)
        want = ref.assign(new, rows)
        check_step(step, want)
        check_tables(cache, ref)
        assert cache._state.tolist()[:2] == [want[3], 0]
        keep = np.where(rng.rand(requests) < 0.3, rng.randint(-1, 3 * page, requests), 1 << 30)
        cache.trim(int32(keep))
        ref.trim(keep)
        check_tables(cache, ref)
    cache.trim([0] * requests)
    assert int(cache.free_count) == cache.pages and sorted(cache.free.tolist()) == list(range(cache.pages))


def test_many_rows_and_pages():
    """Rows and pages of many workgroups, requests without any among them."""
    cache, ref = make(7, 400, 1500, 16, heads=1)
    new = [0, 6000, 1, 0, 5003, 6399, 0]
    step = cache.assign(int32(new), 18000)
    check_step(step, ref.assign(new, 18000))
    check_tables(cache, ref)
    before = cache.free.clone()
    keep = [0, 17, 1, 5, 5002, 0, 0]
    cache.trim(keep)
    ref.trim(keep)
    check_tables(cache, ref)
    # an assign followed by a trim to the old lengths restores the stack
    held, stack = cache.lengths.clone(), cache.free.clone()
    cache.assign(int32([300] * 7), 2100)
    cache.trim(held)
    assert torch.equal(cache.lengths, held) and torch.equal(cache.free, stack) and before.shape == stack.shape


@pytest.mark.parametrize("new,rows,why", [([5, 5, 5], 14, 1), ([97, 0, 0], 97, 2), ([90, 90, 90], 270, 3)])
def test_refused_assign_changes_nothing(new, rows, why):
    import dkv_hip

    cache, ref = make(3, 6, 16, 16)
    cache.assign([20, 1, 0]), ref.assign([20, 1, 0], 21)
    step = cache.assign([n - (20, 1, 0)[i] if n > 20 else n for i, n in enumerate(new)], rows)
    want = ref.assign([n - (20, 1, 0)[i] if n > 20 else n for i, n in enumerate(new)], rows)
    if why == 2:
        step = cache.assign([97 - 20, 0, 0], rows)
        want = ref.assign([97 - 20, 0, 0], rows)
    assert want[3] == why
    check_step(step, want)
    check_tables(cache, ref)
    with pytest.raises(dkv_hip.DkvError, match="nothing was assigned"):
        cache.check()
    cache.assign([1, 1, 1])
    ref.assign([1, 1, 1], 3)
    cache.check()
    check_tables(cache, ref)


def test_no_rows():
    cache, ref = make()
    step = cache.assign([0, 0, 0])
    assert step.rows == 0 and step.cu.tolist() == [0, 0, 0, 0] and step.slots.numel() == 0
    key = torch.empty(0, 2, 64, dtype=torch.float16, device=DEV)
    cache.store(0, key, key, step)
    assert [t.shape[0] for t in cache.load(0, step.slots)] == [0, 0]
    check_tables(cache, ref)


def special_rows(n, heads, dim, seed):
    """Rows whose blocks hold: nothing, ties of every code, one size only, values next to the limits of the exponent."""
    rng = np.random.RandomState(seed)
    x = rng.randn(n, heads, dim)
    flat = x.reshape(-1, 32)
    for i in range(min(len(flat), 40)):
        pick = i % 8
        if pick == 0:
            flat[i] = 0.0
        elif pick == 1:  # the middles between codes, both signs
            flat[i, :14] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0]
            flat[i, 14:] = 6.0
        elif pick == 2:
            flat[i] = 7.0 if i % 16 == 2 else 6.96875  # at and below the step to the next exponent
        elif pick == 3:
            flat[i] *= 2.0 ** -24
        elif pick == 4:
            flat[i] = np.clip(flat[i] * 20000.0, -65504, 65504)
        elif pick == 5:
            flat[i] = 2.0 ** rng.randint(-14, 14, 32) * rng.choice([-1, 1], 32)
        elif pick == 6:
            flat[i] = -0.0
        else:
            flat[i] *= np.where(np.arange(32) == 3, 100.0, 0.01)
    return x


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dim,page", [(1, 64, 16), (3, 64, 64), (2, 128, 32), (1, 256, 16), (5, 128, 16)])
def test_store_and_load(heads, dim, page, dtype):
    print(f"[case] store heads={heads} dim={dim} page={page} {dtype}", flush=True)
    n = 71
    cache, ref = make(2, 8, 20, page, layers=2, heads=heads, dim=dim)
    before = [t.clone() for t in (cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales)]
    step = cache.assign([37, n - 37 - 3], rows=n)  # three rows behind the last request
    t = TYPES[dtype]
    key = torch.tensor(special_rows(n, heads, dim, 1), device=DEV).to(t)
    value = torch.tensor(special_rows(n, heads, dim, 2), device=DEV).to(t)
    # heads before tokens in memory, as attention layers hold them; the values over a wider row
    key = key.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(n, heads, dim + 16, dtype=t, device=DEV)
    wide[..., 8:8 + dim] = value
    value = wide[..., 8:8 + dim]
    cache.store(1, key, value, step)
    assert not cache.key_codes[0].any() and not cache.value_scales[0].any()  # the other layer is left as it was
    for out in TYPES.values():
        got = cache.load(1, step.slots, dtype=out)
        for have, given in zip(got, (key, value)):
            want = paged_ref.quantize(given.double().cpu().numpy())[2]
            want[n - 3:] = 0.0
            assert have.dtype == out and np.array_equal(have.double().cpu().numpy(), want)
    # nothing outside the slots was written
    used = step.slots[:n - 3]
    free = torch.tensor([s for s in range(cache.pages * page) if s not in set(used.tolist())], device=DEV)
    assert not any(t.any() for t in cache.load(1, free, dtype=torch.float32))
    assert all(not b.any() for b in before)


def test_store_overwrites_and_moves_nothing_else():
    """A slot written again holds the new row; its neighbours in the four of tokens keep theirs."""
    cache, _ = make(1, 4, 4, 16, heads=2, dim=128)
    step = cache.assign([21])
    rows = torch.randn(2, 21, 2, 128, device=DEV)
    cache.store(0, rows[0], rows[1], step)
    first = cache.load(0, step.slots, dtype=torch.float32)
    from paged_cache import Step

    one = Step(step.slots[6:7], step.positions[6:7], step.cu, 1, 64, 1)
    again = torch.randn(2, 1, 2, 128, device=DEV) * 9
    cache.store(0, again[0], again[1], one)
    second = cache.load(0, step.slots, dtype=torch.float32)
    for a, b, new in zip(first, second, again):
        want = a.clone()
        want[6] = torch.tensor(paged_ref.quantize(new[0].double().cpu().numpy())[2])
        assert torch.equal(b, want)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_blocks_with_infinities_and_nan(dtype):
    cache, _ = make(1, 4, 4, 16, heads=1, dim=128)
    step = cache.assign([4])
    x = torch.randn(4, 1, 128, device=DEV).to(TYPES[dtype])
    x[0, 0, 5], x[1, 0, 40], x[2, 0, 127] = float("inf"), float("nan"), float("-inf")
    cache.store(0, x, x, step)
    want = paged_ref.quantize(x.double().cpu().numpy())[2]
    for out in TYPES.values():
        for got in cache.load(0, step.slots, dtype=out):
            assert np.array_equal(got.double().cpu().numpy(), want, equal_nan=True)
    assert np.isnan(want).sum() == 3 * 32


def test_float32_extremes():
    """Magnitudes past every fp16: the largest code at the largest exponent, zeros below the smallest step."""
    cache, _ = make(1, 4, 4, 16, heads=1, dim=64)
    step = cache.assign([3])
    x = torch.zeros(3, 1, 64, device=DEV)
    x[0, 0, :3] = torch.tensor([3e38, -1e6, 40000.0])
    x[1, 0, :3] = torch.tensor([1e-45, -3e-39, 1e-30])
    x[2, 0, :4] = torch.tensor([2.0 ** -23, 2.0 ** -24, -(2.0 ** -24) * 1.001, 2.0 ** -22])
    cache.store(0, x, x, step)
    key, value = cache.load(0, step.slots, dtype=torch.float32)
    want = paged_ref.quantize(x.double().cpu().numpy())[2]
    assert np.array_equal(key.double().cpu().numpy(), want) and torch.equal(key, value)
    assert key[0, 0, 0] == 49152 and not key[1].any() and key[2, 0, 0] == 2.0 ** -23 and key[2, 0, 1] == 0


def test_other_stream_and_graph():
    """A step captured once and replayed: pages, slots and rows as the eager steps give them, on a side stream."""
    heads, dim = 2, 64
    cache, ref = make(3, 6, 16, 16, heads=heads, dim=dim)
    new, key, value = int32([1, 1, 1]), torch.randn(3, heads, dim, device=DEV), torch.randn(3, heads, dim, device=DEV)
    cache.assign([15, 3, 0])
    ref.assign([15, 3, 0], 18)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step = cache.assign(new, 3)
        cache.store(0, key, value, step)
    torch.cuda.current_stream().wait_stream(stream)
    check_step(step, ref.assign([1, 1, 1], 3))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = cache.assign(new, 3)
        cache.store(0, key, value, step)
        out = cache.load(0, step.slots, dtype=torch.float32)
    for turn in range(4):
        key.copy_(torch.randn(3, heads, dim, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        check_step(step, ref.assign([1, 1, 1], 3))
        check_tables(cache, ref)
        want = paged_ref.quantize(key.double().cpu().numpy())[2]
        assert np.array_equal(out[0].double().cpu().numpy(), want), turn


def test_past_32_bits():
    """Pages whose bytes lie past 2^32: stored, loaded and attended to like any other."""
    from paged_cache import PagedCache

    heads, dim, page, pages = 8, 256, 4096, 1100
    cache = PagedCache(1, heads, dim, pages, page=page, table_pages=4, device=DEV)
    assert cache.key_codes.numel() > 1 << 32
    cache.free.copy_(torch.arange(pages))  # the last pages first
    step = cache.assign([4100])
    rows = torch.randn(2, 4100, heads, dim, device=DEV)
    cache.store(0, rows[0], rows[1], step)
    assert int(step.slots[0]) == (pages - 1) * page and int(step.slots[-1]) == (pages - 2) * page + 3
    key, value = cache.load(0, step.slots, torch.float32)
    pick = [0, 7, 4095, 4096, 4099]
    for have, given in ((key, rows[0]), (value, rows[1])):
        assert np.array_equal(have[pick].double().cpu().numpy(), paged_ref.quantize(given[pick].double().cpu().numpy())[2])
    query = torch.randn(4100, heads, dim, device=DEV)[-1:].contiguous()
    one = cache.assign([1])
    cache.store(0, rows[0][:1], rows[1][:1], one)
    out = cache.attend_rows(0, query, one)
    weights = torch.softmax(torch.einsum("hd,thd->ht", query[0].double(), torch.cat([key, key[:1]]).double()) * dim ** -0.5, -1)
    want = torch.einsum("ht,thd->hd", weights, torch.cat([value, value[:1]]).double())
    # float32: the weights' error, some 2^-17 (256 products of order 1, 4,101 sums), on values below 8
    assert (out[0].double() - want).abs().max() < 8 * 2.0 ** -17


def page_bytes(cache, arrays, slots, key, value):
    """The cache's four arrays of one layer as include/dimmerkv.h lays them out, after rows went into ``slots``."""
    heads, dim, page = cache.kv_heads, cache.head_dim, cache.page
    key_codes, key_scales, value_codes, value_scales = (a.cpu().numpy().reshape(-1).copy() for a in arrays)
    lane_dims, lane_bytes = dim // 16, dim // 32
    (kc, ks, _), (vc, vs, _) = paged_ref.quantize(key), paged_ref.quantize(value)
    for row, slot in enumerate(slots):
        if slot < 0:
            continue
        p, t = divmod(slot, page)
        for h in range(heads):
            hp = p * heads + h
            for i in range(dim // 2):  # dimension 2i low, 2i + 1 high
                key_codes[(hp * page + t) * (dim // 2) + i] = kc[row, h, 2 * i] | kc[row, h, 2 * i + 1] << 4
                lane, within = divmod(2 * i, lane_dims)
                value_codes[hp * page * (dim // 2) + t // 4 * (2 * dim) + (lane * 4 + t % 4) * lane_bytes + within // 2] = \
                    vc[row, h, 2 * i] | vc[row, h, 2 * i + 1] << 4
            for block in range(dim // 32):
                key_scales[(hp * page + t) * (dim // 32) + block] = ks[row, h, block]
                value_scales[hp * page * (dim // 32) + t // 4 * (dim // 8) + block * 4 + t % 4] = vs[row, h, block]
    return key_codes, key_scales, value_codes, value_scales


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dim,page", [(2, 64, 16), (3, 128, 32), (1, 256, 16), (2, 256, 64)])
def test_stored_bytes(heads, dim, page, dtype):
    """Codes, their signs (of zeros too) and exponents byte by byte where the published form has them, in pages that held
    other bytes, and not a byte outside the slots."""
    print(f"[case] bytes heads={heads} dim={dim} page={page} {dtype}", flush=True)
    n = 43
    cache, _ = make(2, 5, 9, page, layers=2, heads=heads, dim=dim)
    cache.free.copy_(torch.tensor([4, 7, 0, 8, 2, 6, 1, 3, 5], dtype=torch.int32))
    step = cache.assign([23, n - 23 - 2], rows=n)
    key, value = (torch.tensor(special_rows(n, heads, dim, seed), device=DEV).to(TYPES[dtype]) for seed in (3, 4))
    key[5, 0, 3], value[30, heads - 1, dim - 1] = float("nan"), -float("inf")
    g = torch.Generator(DEV).manual_seed(dim)
    every = (cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales)
    for a in every:
        a.copy_(torch.randint(1, 256, a.shape, generator=g, device=DEV))
    other = [a[0].clone() for a in every]
    want = page_bytes(cache, [a[1] for a in every], step.slots.tolist(), key.double().cpu().numpy(), value.double().cpu().numpy())
    cache.store(1, key, value, step)
    for a, b, expected in zip(every, other, want):
        assert torch.equal(a[0], b) and np.array_equal(a[1].cpu().numpy().reshape(-1), expected)


def test_captured_steps_take_counts_on_the_gpu():
    """Host numbers are refused while a step is captured; the capture goes on, and its replays are right."""
    cache, ref = make(2, 6, 16, 16)
    new, keep = int32([3, 2]), int32([1, 99])
    cache.assign([20, 1]), ref.assign([20, 1], 21)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: cache.assign([3, 2]), lambda: cache.trim([1, 99])):
            with pytest.raises(ValueError, match="captured"):
                call()
        step = cache.assign(new, 5)
        cache.trim(keep)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        check_step(step, ref.assign([3, 2], 5))
        ref.trim([1, 99])
        check_tables(cache, ref)
        cache.assign([1, 0]), ref.assign([1, 0], 1)
    cache.check()
