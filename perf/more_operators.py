"""Raw projections into the paged 4-bit cache, and attention of shaped scores over it, as timed cases.

``append``: a step's keys and values go into the pages with the position rotation applied to the keys on the way, and the
queries come back rotated.  ``shaped``: attention of a step's queries over the pages where scores are capped by a tanh,
get a bias that falls with the distance, share their softmax with a sink, or are masked by ranges of tokens (documents
packed into one request, a prefix that sees itself both ways).

The cache's values: 32 consecutive dimensions of one token and head share a power of two 2^e, and each is a 4-bit code
(sign, then 0, 0.5, 1, 1.5, 2, 3, 4, 6) times it.  Pages of ``page`` tokens hold, per KV head,

- keys: token after token, D / 2 bytes (dimension 2i in the low half of byte i) and D / 32 exponents (byte e + 127),
- values: in fours of tokens; inside a four 16 lanes of D / 16 dimensions, each with its four tokens' D / 32 bytes;
  exponents by [block of 32][token of the four].

``run`` in its plain form is elementary torch in 32 bits, and in 64 where a rotated key is cut to 4 bits: next to the
border of two codes 32 bits would take the wrong one.  ``exact`` is the definition in 64 bits.
"""

import math
import os
import sys
import types

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EXP_MIN, EXP_MAX = -22, 13
REACH = 32768  # positions of the rotation's tables


def listed():
    """The shapes are the two model shapes of this package (8 KV heads: 64 dimensions and 32 query heads, 128 and 24) and
    its largest head, 256, at the lengths of its benchmark."""
    plain = {"window": 0, "cap": 0.0, "slopes": False, "sinks": False, "documents": 0, "prefix": 0}
    return [
        # the new tokens of 64 running requests, out of one projection for queries, keys and values
        {"name": "append-decode", "kind": "append", "rows": 64, "kv_heads": 8, "groups": 4, "dim": 64, "rotary": 64,
         "interleaved": False, "fused": True, "page": 64, "dtype": "f16"},
        # a 16K prompt of one layer
        {"name": "append-prefill", "kind": "append", "rows": 16384, "kv_heads": 8, "groups": 3, "dim": 128, "rotary": 128,
         "interleaved": False, "fused": True, "page": 64, "dtype": "bf16"},
        # a chunk of odd length, half of the dimensions rotated in neighbouring pairs, heads before tokens
        {"name": "append-chunk-pairs", "kind": "append", "rows": 1777, "kv_heads": 2, "groups": 8, "dim": 128,
         "rotary": 64, "interleaved": True, "fused": False, "page": 32, "dtype": "f32"},
        # one token under capped scores over the shortest conversation
        {"name": "cap-1500", "kind": "shaped", "requests": 1, "tokens": 1500, "ragged": False, "new": 1, "kv_heads": 4,
         "groups": 2, "dim": 256, "page": 64, "dtype": "bf16"} | plain | {"cap": 50.0},
        # one token over 16K tokens under a bias that falls with the distance
        {"name": "slopes-16k", "kind": "shaped", "requests": 1, "tokens": 16384, "ragged": False, "new": 1, "kv_heads": 8,
         "groups": 4, "dim": 64, "page": 64, "dtype": "f16"} | plain | {"slopes": True},
        # a ragged batch of 32 conversations of up to 32K tokens, one token each, capped scores
        {"name": "cap-ragged-32", "kind": "shaped", "requests": 32, "tokens": 32768, "ragged": True, "new": 1,
         "kv_heads": 8, "groups": 3, "dim": 128, "page": 64, "dtype": "bf16"} | plain | {"cap": 50.0},
        # five drafted tokens each of eight requests in a layer with a sliding window and sinks
        {"name": "sinks-draft-window", "kind": "shaped", "requests": 8, "tokens": 8192, "ragged": True, "new": 5,
         "kv_heads": 8, "groups": 8, "dim": 64, "page": 32, "dtype": "bf16"} | plain | {"window": 128, "sinks": True},
        # a question of 2,048 tokens over a 16K document, capped scores
        {"name": "cap-question", "kind": "shaped", "requests": 1, "tokens": 16384, "ragged": False, "new": 2048,
         "kv_heads": 8, "groups": 3, "dim": 128, "page": 64, "dtype": "bf16"} | plain | {"cap": 50.0},
        # a prompt of eleven documents in which each sees itself only
        {"name": "documents-8k", "kind": "shaped", "requests": 1, "tokens": 8192, "ragged": False, "new": 8192,
         "kv_heads": 8, "groups": 4, "dim": 64, "page": 64, "dtype": "f16"} | plain | {"documents": 11},
        # two prompts whose prefix (an image's tokens, an instruction) sees all of itself, with a distance bias
        {"name": "prefix-slopes", "kind": "shaped", "requests": 2, "tokens": 4001, "ragged": True, "new": 4001,
         "kv_heads": 4, "groups": 3, "dim": 128, "page": 16, "dtype": "bf16"} | plain | {"slopes": True, "prefix": 1300},
        # a short question in 32 bits under everything at once
        {"name": "all-f32", "kind": "shaped", "requests": 3, "tokens": 2500, "ragged": True, "new": 90, "kv_heads": 2,
         "groups": 5, "dim": 64, "page": 16, "dtype": "f32", "window": 1100, "cap": 30.0, "slopes": True, "sinks": True,
         "documents": 3, "prefix": 0},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dim = rng.choice([64, 64, 128, 128, 256])
    if rng.random() < 0.35:
        return {"kind": "append", "rows": _log(rng, 1, 12000), "kv_heads": rng.choice([1, 2, 3, 5, 8] if dim < 256 else [1, 2, 4]),
                "groups": rng.choice([1, 2, 3, 4]), "dim": dim, "rotary": rng.choice([dim, dim, dim // 2, 16, 48]),
                "interleaved": rng.random() < 0.4, "fused": rng.random() < 0.6, "page": rng.choice([16, 32, 64, 128]),
                "dtype": rng.choice(["f32", "f16", "bf16", "bf16"])}
    case = {"kind": "shaped", "dim": dim, "page": rng.choice([16, 32, 64, 128]),
            "dtype": rng.choice(["f32", "f16", "bf16", "bf16"])}
    if rng.random() < 0.55:  # single tokens, or a few drafted ones
        requests = _log(rng, 1, 32)
        case.update(requests=requests, tokens=_log(rng, 1, 32768), ragged=requests > 1, new=rng.choice([1, 1, 1, 2, 4, 5]),
                    groups=rng.choice([1, 2, 3, 4, 7, 8, 16, 20]), kv_heads=rng.choice([1, 2, 4, 8] if dim < 256 else [1, 2, 4]))
    else:  # prompts and questions
        requests = _log(rng, 1, 4)
        case.update(requests=requests, tokens=_log(rng, 16, 8192), ragged=requests > 1, new=_log(rng, 2, 1024),
                    groups=rng.choice([1, 2, 3, 4, 5, 8]), kv_heads=rng.choice([1, 2, 4] if dim < 256 else [1, 2]))
    case.update(window=rng.choice([0, 0, 0, _log(rng, 1, 8192)]), cap=rng.choice([0.0, 0.0, 15.0, 30.0, 50.0]),
                slopes=rng.random() < 0.35, sinks=rng.random() < 0.35, documents=0, prefix=0)
    masked = rng.random()
    if masked < 0.25:
        case["documents"] = rng.randint(2, 12)
    elif masked < 0.45:
        case["prefix"] = _log(rng, 1, 2048)
    elif not (case["cap"] or case["slopes"] or case["sinks"]):
        case["cap"] = 50.0
    return case


# ------------------------------------------------------------------ the cases' sizes, from the case alone

def _lengths(case):
    """(tokens before, new tokens) of each request; the plan's numbers, the same for every seed."""
    g = np.random.RandomState(len(str(case)) * 7919 + case["requests"] * 31 + case["new"])
    n = case["requests"]
    new = np.full(n, case["new"]) if not case["ragged"] or case["new"] < 8 else g.randint(1, case["new"] + 1, n)
    total = np.full(n, case["tokens"]) if not case["ragged"] else (case["tokens"] * g.uniform(0.1, 1.0, n)).astype(int)
    if case["ragged"]:
        total[0], new[0] = case["tokens"], case["new"]
    return np.maximum(total - new, 0), new


def _ranges(case):
    """(first, last) token that each row may see, from its documents and prefix; None where the case has neither.  Every
    40th row of a document batch is padding that sees nothing."""
    if not case["documents"] and not case["prefix"]:
        return None, None
    old, new = _lengths(case)
    g = np.random.RandomState(case["tokens"] + 7 * case["documents"])
    first, last = [], []
    for o, n in zip(old.tolist(), new.tolist()):
        place = np.arange(o, o + n)
        if case["documents"]:
            starts = np.unique(np.concatenate([[0], g.randint(0, o + n, case["documents"] - 1)]))
            begin = starts[np.searchsorted(starts, place, side="right") - 1]
            begin[39::40] = o + n
            first.append(begin)
        else:
            last.append(np.maximum(place, case["prefix"] - 1))
    return np.concatenate(first) if first else None, np.concatenate(last) if last else None


def _seen(case):
    """(low, high) token of each row, all masks taken together, its request and its position."""
    old, new = _lengths(case)
    first, last = _ranges(case)
    owner = np.repeat(np.arange(len(old)), new)
    place = np.concatenate([np.arange(o, o + n) for o, n in zip(old, new)])
    low = np.zeros_like(place) if first is None else first
    if case["window"]:
        low = np.maximum(low, place - case["window"] + 1)
    high = np.minimum(place if last is None else last, (old + new)[owner] - 1)
    return np.maximum(low, 0), high, owner, place


# ------------------------------------------------------------------ the cache's form

def _codes(x):
    """x [..., D] float64 -> 4-bit codes uint8 [..., D] and exponent bytes uint8 [..., D / 32]."""
    blocks = x.unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1)
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 3 + (mantissa >= 0.875).int()
    e = torch.where(amax > 0, e, torch.full_like(e, EXP_MIN)).clamp(EXP_MIN, EXP_MAX)
    size = torch.ldexp(blocks, -e[..., None]).abs().clamp(max=6.0)
    # steps of 0.5 below 2, 1 below 4, 2 above; the place of a size in GRID, ties to the even one
    place = torch.where(size < 2, torch.round(size * 2), torch.where(size < 4, torch.round(size) + 2,
                                                                      torch.round(size * 0.5) + 4)).to(torch.uint8)
    return (place | (torch.signbit(blocks).to(torch.uint8) << 3)).flatten(-2), (e + 127).to(torch.uint8)


def _decode(code, scale):
    """Codes [..., D] and exponent bytes [..., D / 32] -> float32 [..., D]."""
    grid = torch.tensor(GRID, dtype=torch.float32, device=code.device)
    value = grid[(code & 7).long()] * (1.0 - 2.0 * (code >> 3).float())
    power = torch.ldexp(torch.ones((), device=code.device), scale.float() - 127.0)
    return (value.unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)


def _empty_pages(pages, heads, page, dim):
    new = lambda width: torch.zeros(pages + 1, heads, page * width, dtype=torch.uint8, device=DEV)
    return {"key_codes": new(dim // 2), "key_scales": new(dim // 32), "value_codes": new(dim // 2),
            "value_scales": new(dim // 32)}


def _write(pages, slots, key, value, page):
    """Rows [T, H, D] quantized into their slots, in place."""
    heads, dim = key.shape[1:]
    # rows without a slot go to a spare page behind the others
    spare = pages["key_codes"].shape[0] - 1
    where, at = torch.where(slots < 0, torch.full_like(slots, spare), slots // page), slots % page
    code, scale = _codes(key.double())
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    pages["key_codes"].view(-1, heads, page, dim // 2)[where, :, at] = packed
    pages["key_scales"].view(-1, heads, page, dim // 32)[where, :, at] = scale
    code, scale = _codes(value.double())
    packed = (code[..., 0::2] | (code[..., 1::2] << 4)).unflatten(-1, (16, dim // 32))
    pages["value_codes"].view(-1, heads, page // 4, 16, 4, dim // 32)[where, :, at // 4, :, at % 4] = packed
    pages["value_scales"].view(-1, heads, page // 4, dim // 32, 4)[where, :, at // 4, :, at % 4] = scale


def _halves(packed):
    return torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2)


def _rows(pages, slots, heads, page, dim):
    """float32 keys and values [T, H, D] of the slots; zeros where a slot is negative."""
    inside = slots.clamp(min=0)
    where, at = inside // page, inside % page
    key = _decode(_halves(pages["key_codes"].view(-1, heads, page, dim // 2)[where, :, at]),
                  pages["key_scales"].view(-1, heads, page, dim // 32)[where, :, at])
    raw = pages["value_codes"].view(-1, heads, page // 4, 16, 4, dim // 32)[where, :, at // 4, :, at % 4]
    value = _decode(_halves(raw.flatten(-2)),
                    pages["value_scales"].view(-1, heads, page // 4, dim // 32, 4)[where, :, at // 4, :, at % 4])
    gone = (slots < 0)[:, None, None]
    return key.masked_fill(gone, 0.0), value.masked_fill(gone, 0.0)


def _normal(shape, g, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * scale


def _keys(shape, g):
    """Keys as models have them: every channel of its own size, some of them far from zero."""
    heads, dim = shape[-2:]
    size = torch.exp(0.5 * _normal((heads, dim), g))
    offset = _normal((heads, dim), g) * (torch.rand(heads, dim, generator=g, device=DEV) < 0.1)
    return _normal(shape, g) * size + 2.0 * offset


def _tensor(values, dtype):
    return torch.tensor(np.asarray(values), dtype=dtype, device=DEV)


# ------------------------------------------------------------------ inputs

def _inputs(case, seed):
    """What the program has in hand, from the case and the seed."""
    g = torch.Generator(DEV).manual_seed(seed * 1_000_003 + 17)
    host = np.random.RandomState((seed * 7919 + 13) % (1 << 31))
    s = types.SimpleNamespace(case=case, kind=case["kind"])
    heads, dim, page, groups, dtype = case["kv_heads"], case["dim"], case["page"], case["groups"], DTYPES[case["dtype"]]
    if s.kind == "append":
        rows, pairs = case["rows"], case["rotary"] // 2
        s.pages = -(-rows // page) + 3
        used = host.permutation(s.pages)[:-(-rows // page)]
        slots = used[np.arange(rows) // page] * page + np.arange(rows) % page
        # a few requests' tokens, each from its own position on
        parts = np.sort(host.randint(0, rows, 3))
        owner = np.searchsorted(parts, np.arange(rows), side="right")
        begin = np.concatenate([[0], parts])
        start = host.randint(0, REACH - rows, 4)
        positions = start[owner] + np.arange(rows) - begin[owner]
        if rows > 8:
            slots[-2:], positions[-2:] = -1, -1  # a padded batch's rows
        s.slots, s.positions = _tensor(slots, torch.int64), _tensor(positions, torch.int64)
        # the tables, rounded once from 64 bits
        rate = 500000.0 ** (-np.arange(pairs) / pairs)
        angle = np.arange(REACH)[:, None] * rate
        s.cos, s.sin = _tensor(np.cos(angle), torch.float32), _tensor(np.sin(angle), torch.float32)
        query, key = _normal((rows, heads * groups, dim), g, 1.5), _keys((rows, heads, dim), g)
        value = _normal((rows, heads, dim), g)
        if case["fused"]:  # views of one projection's output
            whole = torch.cat([t.flatten(1) for t in (query, key, value)], 1).to(dtype)
            parts = whole.split([heads * groups * dim, heads * dim, heads * dim], 1)
            s.query, s.key, s.value = (t.unflatten(1, (-1, dim)) for t in parts)
        else:  # heads before tokens
            s.query, s.key, s.value = (t.transpose(0, 1).contiguous().to(dtype).transpose(0, 1) for t in (query, key, value))
        return s
    old, new = _lengths(case)
    s.totals, s.new_host = old + new, new
    used = -(-s.totals // page)
    s.pages = int(used.sum()) + 4
    order, at = host.permutation(s.pages), 0
    s.table_host = np.full((len(old), int(used.max()) + 1), -1)
    s.store = _empty_pages(s.pages, heads, page, dim)
    for b, n in enumerate(used):
        s.table_host[b, :n] = order[at:at + n]
        at += n
        tokens = np.arange(int(s.totals[b]))
        slots = _tensor(s.table_host[b, tokens // page] * page + tokens % page, torch.int64)
        _write(s.store, slots, _keys((len(tokens), heads, dim), g), _normal((len(tokens), heads, dim), g), page)
    s.cu_host = np.concatenate([[0], np.cumsum(new)])
    s.rows, s.longest, s.most = int(new.sum()), int(s.totals.max()), int(new.max())
    # scores that reach a cap's bend where there is one
    s.query = _normal((s.rows, heads * groups, dim), g, 3.0 if case["cap"] else 1.5).to(dtype)
    s.table, s.lengths, s.cu = (_tensor(x, torch.int32) for x in (s.table_host, s.totals, s.cu_host))
    s.scaling, s.cap = dim ** -0.5, case["cap"] or None
    q_heads = heads * groups
    s.slopes = _tensor(2.0 ** (-8.0 * np.arange(1, q_heads + 1) / q_heads), torch.float32) if case["slopes"] else None
    s.sinks = _normal((q_heads,), g, 2.0) if case["sinks"] else None
    first, last = _ranges(case)
    s.first = None if first is None else _tensor(first, torch.int64)
    s.last = None if last is None else _tensor(last, torch.int64)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if s.kind == "append":
        s.store = _empty_pages(s.pages, case["kv_heads"], case["page"], case["dim"])
    if not own:
        return s
    for p in (ROOT, os.path.join(ROOT, "dimmer-kv_amd")):
        if p not in sys.path:
            sys.path.insert(0, p)
    import paged_cache

    shaped = s.kind == "shaped"
    s.cache = paged_cache.PagedCache(1, case["kv_heads"], case["dim"], s.pages, page=case["page"],
                                     requests=case["requests"] if shaped else 1,
                                     table_pages=s.table.shape[1] if shaped else s.pages, device=DEV)
    for name in s.store:
        getattr(s.cache, name)[0].copy_(s.store[name][:s.pages])
    del s.store
    if shaped:
        s.cache.table.copy_(s.table)
        s.cache.lengths.copy_(s.lengths)
        s.step = paged_cache.Step(slots=None, positions=None, cu=s.cu, rows=s.rows, longest=s.longest, most=s.most)
    else:
        s.step = paged_cache.Step(slots=s.slots, positions=s.positions, cu=None, rows=case["rows"], longest=0, most=0)
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    return _run_append(s) if s.kind == "append" else _run_shaped(s)


def _turned(x, s):
    """Rows [T, H, D] with their first ``rotary`` dimensions rotated, in the type of ``x``."""
    rotary = s.case["rotary"]
    place = s.positions.clamp(min=0)
    cos, sin = (t[place][:, None].to(x.dtype) for t in (s.cos, s.sin))
    if s.case["interleaved"]:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rotary:]], -1)


def _run_append(s):
    """The queries rotated, and a step's keys (rotated) and values into the cache and out of it again."""
    if own:
        query = s.cache.append(0, s.query, s.key, s.value, s.step, s.cos, s.sin, interleaved=s.case["interleaved"])
        return [query, *s.cache.load(0, s.slots, dtype=s.key.dtype)]
    page, heads, dim = s.case["page"], s.case["kv_heads"], s.case["dim"]
    query = _turned(s.query.float(), s).masked_fill((s.positions < 0)[:, None, None], 0.0).to(s.query.dtype)
    _write(s.store, s.slots, _turned(s.key.double(), s), s.value, page)
    key, value = _rows(s.store, s.slots, heads, page, dim)
    return [query, key.to(s.key.dtype), value.to(s.value.dtype)]


def _run_shaped(s):
    case = s.case
    window = case["window"]
    if own:
        return s.cache.attend_rows(0, s.query, s.step, scaling=s.scaling, window=window or None, cap=s.cap, slopes=s.slopes,
                                   sinks=s.sinks, first=s.first, last=s.last)
    page, heads, dim, groups = case["page"], case["kv_heads"], case["dim"], case["groups"]
    out = torch.empty_like(s.query)
    for b, (total, new) in enumerate(zip(s.totals.tolist(), s.new_host.tolist())):
        at = torch.arange(total, device=DEV)
        key, value = _rows(s.store, s.table[b].long()[at // page] * page + at % page, heads, page, dim)
        begin, end = int(s.cu_host[b]), int(s.cu_host[b + 1])
        query = s.query[begin:end].float().unflatten(1, (heads, groups))
        place = torch.arange(total - new, total, device=DEV)[:, None]
        hidden = at > (place if s.last is None else s.last[begin:end, None])
        if s.first is not None:
            hidden = hidden | (at < s.first[begin:end, None])
        if window:
            hidden = hidden | (at <= place - window)
        for h in range(heads):
            scores = torch.matmul(query[:, h].reshape(new * groups, dim), key[:, h].t().contiguous()) * s.scaling
            scores = scores.view(new, groups, total)
            if s.cap is not None:
                scores = torch.tanh(scores / s.cap) * s.cap
            if s.slopes is not None:
                scores = scores - s.slopes[h * groups:(h + 1) * groups, None] * (place - at).abs().float()[:, None]
            scores = scores.masked_fill(hidden[:, None], float("-inf"))
            highest = scores.amax(-1, keepdim=True)
            if s.sinks is not None:
                sink = s.sinks[h * groups:(h + 1) * groups, None]
                highest = torch.maximum(highest, sink)
            highest = highest.masked_fill(highest == float("-inf"), 0.0)  # a row that sees nothing
            scores = torch.exp(scores - highest)
            whole = scores.sum(-1, keepdim=True)
            if s.sinks is not None:
                whole = whole + torch.exp(sink - highest)
            mixed = torch.matmul(scores.view(new * groups, total), value[:, h]).view(new, groups, dim)
            mixed = mixed / whole.masked_fill(whole == 0.0, 1.0)
            out[begin:end, h * groups:(h + 1) * groups] = mixed.to(out.dtype)
    return out


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    heads, dim, groups = case["kv_heads"], case["dim"], case["groups"]
    element = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["kind"] == "append":
        values, queries = 2 * case["rows"] * heads * dim, case["rows"] * heads * groups * dim
        # queries in and out; keys and values in, their codes written and read, out; a row's angles, slot and position
        return {"bytes": int(2 * queries * element + values * (2 * element + 2 * (0.5 + 1 / 32)))
                + case["rows"] * (4 * case["rotary"] + 16),
                "flops": 3 * case["rows"] * case["rotary"] * heads * (groups + 1) + 3 * values}
    low, high, owner, _ = _seen(case)
    pairs = int(np.maximum(high - low + 1, 0).sum())
    tokens = 0
    for b in range(case["requests"]):  # tokens that some row of the request sees
        begin, end = low[owner == b], high[owner == b] + 1
        begin, end = begin[begin < end], end[begin < end]
        edge = np.zeros(int(end.max()) + 1 if len(end) else 1, np.int64)
        np.add.at(edge, begin, 1)
        np.add.at(edge, end, -1)
        tokens += int((np.cumsum(edge) > 0).sum())
    rows = len(owner)
    ranges = 8 * rows * ((case["documents"] > 0) + (case["prefix"] > 0))
    return {"bytes": int(2 * tokens * heads * dim * (0.5 + 1 / 32)) + 2 * rows * heads * groups * dim * element + ranges,
            "flops": 4 * pairs * heads * groups * dim}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_append(s) if s.kind == "append" else _exact_shaped(s)


def _nearest(x):
    """Each value of x [..., D] as the cache holds it, by trying every code."""
    blocks = x.double().unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1, keepdim=True)
    low = torch.floor(torch.log2(amax.clamp(min=2.0 ** -60)))
    low = torch.where(2.0 ** low > amax, low - 1, torch.where(2.0 ** (low + 1) <= amax, low + 1, low))
    unit = 2.0 ** torch.clamp(low - 2 + (amax >= 1.75 * 2.0 ** low).double(), EXP_MIN, EXP_MAX)
    size = blocks.abs() / unit
    best = torch.zeros_like(size)
    for i, (a, b) in enumerate(zip(GRID, GRID[1:])):
        middle = (a + b) / 2
        # a tie goes to the code of the even place
        up = size >= middle if i % 2 else size > middle
        best = torch.where(up, torch.full_like(best, b), best)
    return (torch.sign(blocks) * best * unit).flatten(-2)


def _exact_append(s):
    """The rotation as a product of complex numbers, pair by pair."""
    case, pairs = s.case, s.case["rotary"] // 2
    along = torch.arange(pairs, device=DEV)
    one, two = (2 * along, 2 * along + 1) if case["interleaved"] else (along, along + pairs)
    place = s.positions.clamp(min=0)
    factor = torch.complex(s.cos.double()[place], s.sin.double()[place])[:, None]

    def rotated(x):
        x = x.double().contiguous().clone()
        z = torch.complex(x[..., one], x[..., two]) * factor
        x[..., one], x[..., two] = z.real, z.imag
        return x

    gone = (s.slots < 0)[:, None, None]
    return [rotated(s.query).masked_fill(gone, 0.0), _nearest(rotated(s.key)).masked_fill(gone, 0.0),
            _nearest(s.value).masked_fill(gone, 0.0)]


def _unpacked(s, b, head):
    """float64 keys and values [total, D] of one request's head, byte by byte of its pages."""
    page, dim = s.case["page"], s.case["dim"]
    total = int(s.totals[b])
    ids = torch.tensor(s.table_host[b, :-(-total // page)], device=DEV)
    signed = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device=DEV)

    def values(raw):
        return torch.stack([signed[(raw & 15).long()], signed[(raw >> 4).long()]], -1).flatten(-2)

    key = values(s.store["key_codes"][ids, head].view(-1, dim // 2))
    key = key.view(-1, dim // 32, 32) * 2.0 ** (s.store["key_scales"][ids, head].view(-1, dim // 32, 1).double() - 127)
    raw = s.store["value_codes"][ids, head].view(-1, 16, 4, dim // 32).permute(0, 2, 1, 3).reshape(-1, dim // 2)
    power = s.store["value_scales"][ids, head].view(-1, dim // 32, 4).permute(0, 2, 1).reshape(-1, dim // 32, 1)
    value = values(raw).view(-1, dim // 32, 32) * 2.0 ** (power.double() - 127)
    return key.reshape(-1, dim)[:total], value.reshape(-1, dim)[:total]


def _exact_shaped(s):
    case = s.case
    heads, groups = case["kv_heads"], case["groups"]
    low, high, _, place = _seen(case)
    low, high, place = (torch.tensor(a, device=DEV)[:, None] for a in (low, high, place))
    out = torch.zeros(s.query.shape, dtype=torch.float64, device=DEV)
    for b in range(case["requests"]):
        total, begin, end = int(s.totals[b]), int(s.cu_host[b]), int(s.cu_host[b + 1])
        at = torch.arange(total, device=DEV)[None]
        for h in range(heads):
            key, value = _unpacked(s, b, h)
            for g in range(h * groups, (h + 1) * groups):
                for lo in range(begin, end, 1024):
                    hi = min(end, lo + 1024)
                    logit = s.query[lo:hi, g].double() @ key.t().contiguous() * s.scaling
                    if s.cap is not None:
                        logit = s.cap * torch.tanh(logit / s.cap)
                    if s.slopes is not None:
                        logit = logit - s.slopes[g].double() * (at - place[lo:hi]).abs()
                    visible = (at >= low[lo:hi]) & (at <= high[lo:hi])
                    logit = torch.where(visible, logit, torch.full_like(logit, -math.inf))
                    # the sink as one more token whose value is nothing
                    sink = torch.full_like(logit[:, :1], -math.inf if s.sinks is None else float(s.sinks[g]))
                    weight = torch.softmax(torch.cat([logit, sink], 1), -1)[:, :-1]
                    out[lo:hi, g] = torch.nan_to_num(weight) @ value
    return out
