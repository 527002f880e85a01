"""The paged 4-bit cache's refusals, before anything is launched (no GPU needed), and its oracle against closed forms."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import dkv_hip
from oracle import paged_ref

P = 64  # a stand-in for a device pointer: 16-byte aligned and never read here


def pages(**change):
    fields = dict(lengths=P, table=P, free_pages=P, free_count=P, state=P, requests=3, width=4, page=16, pages=12)
    fields.update(change)
    return dkv_hip.Pages(**fields)


def cache(**change):
    fields = dict(key_codes=P, key_scales=P, value_codes=P, value_scales=P, pages=4, kv_heads=2, page=16, head_dim=64)
    fields.update(change)
    return dkv_hip.Fp4Cache(**fields)


def refused(rc, code, words):
    assert rc == code and words in dkv_hip.lib().dkv_last_error().decode()


def assign(p, new=P, rows=4, slots=P, positions=P, cu=P):
    return dkv_hip.lib().dkv_page_assign(None if p is None else ctypes.addressof(p), new, rows, slots, positions, cu, None)


@pytest.mark.parametrize("change,code,words", [
    (dict(requests=0), -2, "bad shape"), (dict(requests=8193), -2, "at most 8192"), (dict(width=0), -2, "bad shape"),
    (dict(pages=-1), -2, "bad shape"), (dict(page=8), -2, "power of two"), (dict(page=48), -2, "power of two"),
    (dict(page=8192), -2, "power of two"), (dict(page=4096, width=1 << 19), -2, "2^31"),
    (dict(lengths=None), -1, "null"), (dict(table=None), -1, "null"), (dict(free_pages=None), -1, "null"),
    (dict(free_count=None), -1, "null"), (dict(state=None), -1, "null")])
def test_page_tables_refused(change, code, words):
    p = pages(**change)
    refused(assign(p), code, words)
    refused(dkv_hip.lib().dkv_page_trim(ctypes.addressof(p), P, None), code, words)


def test_page_calls_refused():
    refused(assign(None), -1, "null pages")
    refused(assign(pages(), rows=-1), -2, "-1 rows")
    for name in ("new", "slots", "positions", "cu"):
        refused(assign(pages(), **{name: None}), -1, "null pointer")
    p = pages()
    refused(dkv_hip.lib().dkv_page_trim(ctypes.addressof(p), None, None), -1, "null pointer")


def store(c, key=P, value=P, dtype=1, strides=(128, 64, 128, 64), slots=P, n=5):
    return dkv_hip.lib().dkv_fp4_store(None if c is None else ctypes.addressof(c), key, value, dtype, *strides, slots, n, None)


@pytest.mark.parametrize("change,code,words", [
    (dict(key_codes=None), -1, "null cache"), (dict(value_scales=None), -1, "null cache"), (dict(value_codes=72), -1, "aligned"),
    (dict(key_scales=65), -1, "aligned"), (dict(head_dim=96), -2, "head_dim"), (dict(head_dim=32), -2, "head_dim"),
    (dict(pages=0), -2, "bad cache"), (dict(kv_heads=0), -2, "bad cache"), (dict(kv_heads=65536), -2, "bad cache"),
    (dict(page=24), -2, "bad cache")])
def test_caches_refused(change, code, words):
    c = cache(**change)
    refused(store(c), code, words)
    refused(dkv_hip.lib().dkv_fp4_load(ctypes.addressof(c), P, 5, P, P, 1, None), code, words)


def test_rows_refused():
    refused(store(None), -1, "null cache")
    refused(store(cache(), dtype=3), -1, "dtype 3")
    refused(store(cache(), n=-1), -2, "-1 rows")
    for name in ("key", "value", "slots"):
        refused(store(cache(), **{name: None}), -1, "null pointer")
    refused(store(cache(), key=72), -1, "aligned")
    refused(store(cache(), strides=(128, 60, 128, 64)), -1, "multiples")
    refused(store(cache(), dtype=0, strides=(128, 62, 128, 64)), -1, "multiples")
    assert store(cache(), key=None, n=0) == 0  # nothing to do


def test_python_refusals():
    from paged_cache import PagedCache

    for bad in (dict(head_dim=96), dict(page=24), dict(page=8), dict(pages=0), dict(requests=0), dict(requests=9000),
                dict(kv_heads=0), dict(table_pages=1 << 26), dict(device="cpu")):
        kwargs = dict(layers=1, kv_heads=2, head_dim=64, pages=4, page=64, device="cuda") | bad
        with pytest.raises(ValueError):
            PagedCache(**kwargs)
    rows, slots = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int64)
    for key, value, where in ((rows, rows, slots), (rows.double(), rows.double(), slots), (rows, rows.half(), slots),
                              (rows[:, :1], rows, slots), (rows, rows, slots.int()), (rows[:2], rows[:2], slots)):
        with pytest.raises(ValueError):
            dkv_hip.fp4_store(cache(), key, value, where)
    for keep in (torch.zeros(3, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)):
        with pytest.raises(ValueError):
            dkv_hip.page_trim(pages(), keep)


def test_oracle_quantize():
    grid = np.concatenate([paged_ref.GRID, -paged_ref.GRID])
    for e in (-22, -3, 0, 13):
        row = np.resize(grid, 32) * 2.0 ** e
        assert np.array_equal(paged_ref.quantize(row)[2], row)  # the cache's own values stay
        assert paged_ref.quantize(row)[1].tolist() == [e + 127]
    rng = np.random.RandomState(0)
    x = rng.randn(50, 64) * np.exp(rng.randn(50, 1) * 3)
    codes, scales, values = paged_ref.quantize(x)
    unit = np.repeat(2.0 ** (scales.astype(float) - 127), 32, axis=-1)
    # half a step of the largest codes (4 to 6), but for what lies between 6 and 7 units
    assert (np.abs(values - x) <= unit * 1.0).all() and np.abs(x / unit).max() < 7.0
    assert (codes >> 3 == np.signbit(x)).all()


def test_oracle_attend_against_softmax():
    rng = np.random.RandomState(1)
    q, k, v = rng.randn(4, 6, 8), rng.randn(9, 2, 8), rng.randn(9, 2, 8)
    want = torch.nn.functional.scaled_dot_product_attention(
        torch.tensor(q).transpose(0, 1), torch.tensor(k).transpose(0, 1).repeat_interleave(3, 0),
        torch.tensor(v).transpose(0, 1).repeat_interleave(3, 0),
        attn_mask=torch.ones(4, 9).tril(5).bool(), scale=0.3).transpose(0, 1).numpy()
    assert np.allclose(paged_ref.attend(q, k, v, 0.3), want, atol=1e-12)
    assert not paged_ref.attend(q[:1], k[:0], v[:0], 0.3).any()


def test_oracle_tables():
    t = paged_ref.Tables(2, 3, 5, 16)
    assert t.assign([17, 1], 20)[0] == [0 * 16 + i for i in range(16)] + [16, 32, -1, -1] and t.free == [4, 3]
    t.trim([16, 1])
    assert t.free == [4, 3, 1] and t.table == [[0], [2]]
    assert t.assign([33, 0], 33)[3] == 2 and t.assign([32, 33], 65)[3] == 3 and t.lengths == [16, 1]


def attend_args(**change):
    a = dkv_hip.Fp4AttendArgs()
    fields = dict(cache=cache(), table=P, lengths=P, cu=P, query=P, out=P, query_token=256, query_head=64, requests=2,
                  width=4, rows=3, q_heads=4, query_dtype=2, window=0, longest=64, most=2, scaling=0.125, fill=0)
    fields.update(change)
    for name, value in fields.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,code,words", [
    (dict(cache=cache(head_dim=80)), -2, "head_dim"), (dict(cache=cache(page=20)), -2, "bad cache"),
    (dict(cache=cache(key_codes=None)), -1, "null cache"), (dict(query_dtype=5), -1, "dtype 5"),
    (dict(requests=0), -2, "bad shape"), (dict(requests=8193), -2, "bad shape"), (dict(width=0), -2, "bad shape"),
    (dict(width=1 << 27), -2, "bad shape"), (dict(rows=-1), -2, "bad shape"), (dict(q_heads=3), -2, "3 query heads"),
    (dict(q_heads=0), -2, "query heads"), (dict(rows=1 << 30), -2, "2^31"), (dict(window=-1), -2, "window"),
    (dict(table=None), -1, "null pointer"), (dict(lengths=None), -1, "null pointer"), (dict(cu=None), -1, "null pointer"),
    (dict(query=None), -1, "null pointer"), (dict(out=None), -1, "null pointer"), (dict(query=72), -1, "aligned"),
    (dict(out=72), -1, "aligned"), (dict(query_token=100), -1, "aligned"), (dict(query_dtype=0, query_head=66), -1, "aligned")])
def test_attention_refused(change, code, words):
    a = attend_args(**change)
    refused(dkv_hip.lib().dkv_fp4_attend(ctypes.addressof(a), P, 1 << 20, None), code, words)


def test_attention_workspace():
    lib = dkv_hip.lib()
    lib.dkv_fp4_attend_workspace_bytes.restype = ctypes.c_size_t
    bad = attend_args(q_heads=3)
    assert lib.dkv_fp4_attend_workspace_bytes(ctypes.addressof(bad)) == 0
    long = attend_args(longest=1 << 16, rows=1, most=1, requests=1)
    need = lib.dkv_fp4_attend_workspace_bytes(ctypes.addressof(long))
    assert need > 16
    refused(lib.dkv_fp4_attend(ctypes.addressof(long), P, 16, None), -3, "workspace")
    refused(lib.dkv_fp4_attend(ctypes.addressof(long), None, need, None), -1, "workspace")
    refused(lib.dkv_fp4_attend(ctypes.addressof(long), 72, need, None), -1, "aligned")
    none = attend_args(rows=0)
    assert lib.dkv_fp4_attend(ctypes.addressof(none), None, 0, None) == 0
    refused(lib.dkv_fp4_attend(None, None, 0, None), -1, "null arguments")


def test_most_rows():
    c = cache()
    for call in (store(c, n=2**31 - 1), dkv_hip.lib().dkv_fp4_load(ctypes.addressof(c), P, 2**31 - 1, P, P, 1, None)):
        refused(call, -2, "2147483647 rows")
    refused(assign(pages(), rows=2**31 - 1), -2, "2147483647 rows")


@pytest.mark.parametrize("family,words", [("Gemma2", "soft cap"), ("GptOss", "sinks")])
def test_attention_of_more_than_scores_is_refused(family, words):
    """Models whose attention has a soft cap or sinks, before anything is stored; without them such a model is taken (as far
    as the GPU that this test does without)."""
    import transformers
    from paged_cache import PagedContext

    sizes = dict(num_hidden_layers=2, hidden_size=64, intermediate_size=64, num_attention_heads=2, num_key_value_heads=1,
                 head_dim=64, vocab_size=50)
    if family == "GptOss":
        sizes |= dict(num_local_experts=2, num_experts_per_tok=1)
    config = getattr(transformers, f"{family}Config")(**sizes)
    model = getattr(transformers, f"{family}ForCausalLM")(config)
    caches = [torch.zeros(1, 1, 5, 64) for _ in range(2)]
    with pytest.raises(ValueError, match=words):
        PagedContext(caches, caches, model)
    config.attn_logit_softcapping = None
    for module in model.modules():
        if hasattr(module, "sinks"):
            module.sinks = None
    with pytest.raises(ValueError, match="needs a GPU"):
        PagedContext(caches, caches, model)


def host_cache(**change):
    """A PagedCache's tables on the CPU, for what is decided before any kernel."""
    from paged_cache import PagedCache

    c = PagedCache.__new__(PagedCache)
    fields = dict(device=torch.device("cpu"), requests=2, table_pages=3, page=16, layers=1, kv_heads=2, head_dim=64,
                  table=torch.tensor([[4, 2, -1], [0, -1, -1]], dtype=torch.int32))
    for name, value in (fields | change).items():
        setattr(c, name, value)
    return c


def test_slots_past_the_table_are_refused():
    c = host_cache()
    assert c.slots(0, 14, 18).tolist() == [78, 79, 32, 33] and c.slots(1, 48, 48).numel() == 0
    for start, stop in ((0, 49), (-1, 5), (5, 4), (48, 64)):
        with pytest.raises(ValueError, match="slots"):
            c.slots(0, start, stop)


def test_trim_refuses_counts_of_another_device(monkeypatch):
    """The tables' GPU is the one to launch on; counts that lie elsewhere would be launched on theirs."""
    launched = []
    monkeypatch.setattr(dkv_hip, "page_trim", lambda pages, keep: launched.append(keep))
    c = host_cache(_pages=None)
    with pytest.raises(ValueError, match="trim: tensors must be on"):
        c.trim(torch.zeros(2, dtype=torch.int32, device="meta"))
    assert not launched
    c.trim([1, 0])
    assert launched[0].tolist() == [1, 0] and launched[0].dtype == torch.int32


def test_queries_under_the_result():
    """Whether a result lies over queries other than in their place."""
    size, heads, dim = 4, 2, 64

    def meets(query, out):
        a = dkv_hip.Fp4AttendArgs()
        a.query, a.query_token, a.query_head = query.data_ptr(), query.stride(0), query.stride(1)
        return dkv_hip._query_meets(query, a, out)

    room = torch.zeros(12 * heads * dim)
    rows = lambda first, n=4: room[first * heads * dim:(first + n) * heads * dim].view(n, heads, dim)
    assert not meets(rows(2), rows(2)) and not meets(rows(0), rows(4)) and not meets(rows(4), rows(0))
    assert meets(rows(2), rows(3)) and meets(rows(3), rows(2))
    apart = room[:8 * heads * dim].view(4, 2, heads, dim)[:, 0]  # every second row
    assert meets(apart, rows(0)) and meets(apart, rows(5)) and not meets(apart, rows(7))
    assert not meets(apart[:2], rows(3, 2)) and not meets(apart[:2, :1], room[dim:dim * 3].view(2, 1, dim))
    swapped = rows(0).view(heads, 4, dim).transpose(0, 1)  # heads before rows at the same address
    assert meets(swapped, rows(0))


def test_arrival_words_suffice():
    """More words than a cache has make no other launch: its splits, as the workspace tells, are the same with 2^20."""
    from paged_cache import ARRIVAL_WORDS

    need = dkv_hip.lib().dkv_fp4_attend_workspace_bytes
    splits = set()
    for dim in (64, 128, 256):
        for dtype in (0, 1, 2):
            for requests, heads, groups in ((1, 1, 1), (1, 8, 4), (16, 8, 3), (32, 8, 1), (60, 4, 2), (300, 1, 7), (8192, 8, 1)):
                for longest in (100, 1500, 6000, 40000, 1 << 20):
                    for most in (1, 3, 9):
                        sizes = [need(ctypes.addressof(attend_args(
                            cache=cache(head_dim=dim, kv_heads=heads), requests=requests, q_heads=heads * groups, longest=longest,
                            width=1 << 17, most=most, rows=requests * most, query_dtype=dtype, arrivals=P, arrivals_count=count)))
                            for count in (ARRIVAL_WORDS, 1 << 20)]
                        assert sizes[0] == sizes[1] >= 16
                        splits.add((sizes[0] - 16) // (requests * most * heads * groups * (dim + 2) * 4))
    assert len(splits) > 10


def test_arrival_words_held(monkeypatch):
    """The words of a cache do not grow with its requests (they took 134 MB at 8,192 requests of 8 KV heads)."""
    import paged_cache

    for name in ("zeros", "full", "arange"):  # what a cache allocates, on no device
        make = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda *a, make=make, **k: make(*a, **(k | {"device": "meta"})))
    c = paged_cache.PagedCache(1, 8, 64, 16, requests=8192, table_pages=4, device="cuda")
    assert c._arrivals.numel() * 4 <= 1 << 18
    assert c.held_bytes() == sum(t.numel() * t.element_size() for t in (
        c.key_codes, c.key_scales, c.value_codes, c.value_scales, c.table, c.lengths, c.free, c.free_count, c._state, c._arrivals))


def test_counts_of_other_requests_are_refused():
    import paged_cache

    c = host_cache(_pages=pages(requests=2))
    for new in ([], [1], [1, 2, 3]):
        with pytest.raises(ValueError):
            paged_cache.PagedCache.assign(c, new)
        with pytest.raises(ValueError):
            c.trim(new)


def test_host_numbers_in_a_captured_step_are_refused(monkeypatch):
    """A graph would hold the copy from host memory that is given back after the call."""
    copies = []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(dkv_hip, "to_device", lambda *a: copies.append(a))
    monkeypatch.setattr(dkv_hip, "page_trim", lambda *a: None)
    c = host_cache(device=torch.device("cuda", 0), _pages=None)
    with pytest.raises(ValueError, match="captured"):
        c.trim([1, 0])
    assert not copies
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    c.trim([1, 0])
    assert len(copies) == 1
