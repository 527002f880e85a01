"""The paged 4-bit cache and the reply controls, as timed cases.

One decode step of a serving loop is: pages for the new tokens (``pages``), their keys and values into the cache and,
where a prefix is used again, back out of it (``store``), attention of the queries over the cache (``attend``), and
the logits of the reply under penalties, biases and a grammar with the token picked (``logits``).

The cache's values: 32 consecutive dimensions of one token and head share a power of two 2^e, and each is a 4-bit code
(sign, then 0, 0.5, 1, 1.5, 2, 3, 4, 6) times it.  Pages of ``page`` tokens hold, per KV head,

- keys: token after token, D / 2 bytes (dimension 2i in the low half of byte i) and D / 32 exponents (byte e + 127),
- values: in fours of tokens; inside a four 16 lanes of D / 16 dimensions, each with its four tokens' D / 32 bytes;
  exponents by [block of 32][token of the four].

``run`` in its plain form is elementary torch in 32 bits, ``exact`` the definition in 64 bits.
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
EXP_MIN, EXP_MAX, EXP_NAN = -22, 13, 255


def listed():
    """The shapes are the two model shapes of this package (8 KV heads: 64 dimensions and 32 query heads, 128 and 24),
    at the lengths of its benchmark, and a vocabulary of 128,256."""
    return [
        # one more token for each of 256 running requests: the slot map of a decode step
        {"name": "pages-decode", "kind": "pages", "requests": 256, "page": 64, "longest": 16384, "new": 1},
        # 48 prompts admitted at once, ragged: the slot map of a batched prefill
        {"name": "pages-admit", "kind": "pages", "requests": 48, "page": 64, "longest": 1, "new": 8192},
        # the new token of 64 requests into the cache
        {"name": "store-decode", "kind": "store", "rows": 64, "kv_heads": 8, "dim": 64, "page": 64, "dtype": "f16"},
        # a 16K prompt's keys and values of one layer into the cache, and out again for a request that shares them
        {"name": "store-prefill", "kind": "store", "rows": 16384, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16"},
        # one token over the shortest conversation, float32 queries
        {"name": "attend-1b-1500", "kind": "attend", "requests": 1, "tokens": 1500, "ragged": False, "new": 1,
         "kv_heads": 8, "groups": 4, "dim": 64, "page": 16, "window": 0, "dtype": "f32"},
        # one token over 16K tokens
        {"name": "attend-3b-16k", "kind": "attend", "requests": 1, "tokens": 16384, "ragged": False, "new": 1,
         "kv_heads": 8, "groups": 3, "dim": 128, "page": 64, "window": 0, "dtype": "bf16"},
        # a ragged batch of 32 conversations of up to 32K tokens, one token each
        {"name": "attend-3b-ragged-32", "kind": "attend", "requests": 32, "tokens": 32768, "ragged": True, "new": 1,
         "kv_heads": 8, "groups": 3, "dim": 128, "page": 64, "window": 0, "dtype": "bf16"},
        # five drafted tokens each of eight requests, checked at once under a sliding window
        {"name": "attend-draft-window", "kind": "attend", "requests": 8, "tokens": 8192, "ragged": True, "new": 5,
         "kv_heads": 8, "groups": 4, "dim": 64, "page": 32, "window": 4096, "dtype": "f16"},
        # a question of 2,048 tokens over a 16K document
        {"name": "attend-3b-question", "kind": "attend", "requests": 1, "tokens": 16384, "ragged": False, "new": 2048,
         "kv_heads": 8, "groups": 3, "dim": 128, "page": 64, "window": 0, "dtype": "bf16"},
        # the logits of one reply after a 1,500-token conversation
        {"name": "logits-1", "kind": "logits", "rows": 1, "vocab": 128256, "history": 1500, "biased": 0,
         "masked": False, "dtype": "f32"},
        # the logits of 128 replies: histories of up to 16K tokens, biases, every second one under a grammar
        {"name": "logits-128", "kind": "logits", "rows": 128, "vocab": 128256, "history": 16384, "biased": 64,
         "masked": True, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["pages", "store", "attend", "attend", "attend", "logits"])
    if kind == "pages":
        if rng.random() < 0.5:  # running requests take a few tokens each
            return {"kind": kind, "requests": _log(rng, 1, 1024), "page": rng.choice([16, 32, 64, 128]),
                    "longest": _log(rng, 1, 16384), "new": rng.randint(1, 6)}
        return {"kind": kind, "requests": _log(rng, 1, 48), "page": rng.choice([16, 32, 64, 128]),
                "longest": _log(rng, 1, 2048), "new": _log(rng, 2, 8192)}
    if kind == "store":
        return {"kind": kind, "rows": _log(rng, 1, 16384), "kv_heads": rng.choice([1, 2, 3, 5, 8]),
                "dim": rng.choice([64, 64, 128, 128, 256]), "page": rng.choice([16, 32, 64, 128]),
                "dtype": rng.choice(["f32", "f16", "bf16"])}
    if kind == "logits":
        rows = _log(rng, 1, 128)
        return {"kind": kind, "rows": rows, "vocab": rng.choice([256, 32000, 50257, 128256, _log(rng, 100, 128256)]),
                "history": _log(rng, 1, 16384), "biased": rng.choice([0, 1, 7, 64, 300]),
                "masked": rng.random() < 0.5, "dtype": rng.choice(["f32", "f16", "bf16"])}
    dim = rng.choice([64, 64, 128, 128, 256])
    shape = {"kind": kind, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
             "dtype": rng.choice(["f32", "f16", "bf16", "bf16"])}
    if rng.random() < 0.6:  # single tokens, or a few drafted ones
        requests = _log(rng, 1, 32)
        shape.update(requests=requests, tokens=_log(rng, 1, 32768), ragged=requests > 1,
                     new=rng.choice([1, 1, 1, 2, 4, 5]), groups=rng.choice([1, 2, 3, 4, 7, 8, 16, 20]),
                     kv_heads=rng.choice([1, 2, 4, 8] if dim < 256 else [1, 2, 4]))
    else:  # prompts and questions
        requests = _log(rng, 1, 4)
        shape.update(requests=requests, tokens=_log(rng, 16, 8192), ragged=requests > 1, new=_log(rng, 2, 1024),
                     groups=rng.choice([1, 2, 3, 4, 5, 8]), kv_heads=rng.choice([1, 2, 4] if dim < 256 else [1, 2]))
    shape["window"] = rng.choice([0, 0, 0, _log(rng, 1, 8192)])
    return shape


# ------------------------------------------------------------------ the cases' sizes, from the case alone

def _lengths(case):
    """(tokens before, new tokens) of each request; the plan's numbers, the same for every seed."""
    g = np.random.RandomState(len(str(case)) * 7919 + case["requests"] * 31 + case["new"])
    n = case["requests"]
    if case["kind"] == "pages":
        old = g.randint(0, case["longest"], n) if case["longest"] > 1 else np.zeros(n, int)
        new = np.ones(n, int) if case["new"] == 1 else g.randint(max(1, case["new"] // 8), case["new"] + 1, n)
        if n > 2 and case["new"] != 1:
            new[g.randint(0, n)] = 0  # a request that gets none
        return old, new
    new = np.full(n, case["new"]) if not case["ragged"] or case["new"] < 8 else g.randint(1, case["new"] + 1, n)
    total = np.full(n, case["tokens"]) if not case["ragged"] else (case["tokens"] * g.uniform(0.1, 1.0, n)).astype(int)
    if case["ragged"]:
        total[0] = case["tokens"]
    return np.maximum(total - new, 0), new


def _history(case):
    """Tokens in each row's history and how many of them are its prompt's."""
    g = np.random.RandomState(case["rows"] * 131 + case["history"])
    length = np.array([case["history"]] + [int(case["history"] * u) for u in g.uniform(0.0, 1.0, case["rows"] - 1)])
    return length, (length * g.uniform(0.3, 1.0, case["rows"])).astype(int)


# ------------------------------------------------------------------ the cache's form

def _codes(x):
    """x [..., D] -> 4-bit codes uint8 [..., D] and exponent bytes uint8 [..., D / 32]."""
    blocks = x.float().unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1)
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 3 + (mantissa >= 0.875).int()
    e = torch.where(amax > 0, e, torch.full_like(e, EXP_MIN)).clamp(EXP_MIN, EXP_MAX)
    bad = ~torch.isfinite(blocks).all(-1)
    a = torch.ldexp(blocks, -e[..., None].float())
    size = a.abs().clamp(max=6.0)
    # steps of 0.5 below 2, 1 below 4, 2 above; the place of a size in GRID
    place = torch.where(size < 2, torch.round(size * 2), torch.where(size < 4, torch.round(size) + 2,
                                                                      torch.round(size * 0.5) + 4))
    place = torch.nan_to_num(place).to(torch.uint8)
    code = torch.where(bad[..., None], torch.zeros_like(place), place | (torch.signbit(blocks).to(torch.uint8) << 3))
    scale = torch.where(bad, torch.full_like(e, EXP_NAN), e + 127).to(torch.uint8)
    return code.flatten(-2), scale


def _decode(code, scale):
    """Codes [..., D] and exponent bytes [..., D / 32] -> float32 [..., D]."""
    grid = torch.tensor(GRID, dtype=torch.float32, device=code.device)
    value = grid[(code & 7).long()] * (1.0 - 2.0 * (code >> 3).float())
    power = torch.ldexp(torch.ones((), device=code.device), scale.float() - 127.0)
    power = torch.where(scale == EXP_NAN, torch.full_like(power, float("nan")), power)
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
    code, scale = _codes(key)
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    pages["key_codes"].view(-1, heads, page, dim // 2)[where, :, at] = packed
    pages["key_scales"].view(-1, heads, page, dim // 32)[where, :, at] = scale
    code, scale = _codes(value)
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


def _int32(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ inputs

def _inputs(case, seed):
    """What the program has in hand, from the case and the seed."""
    g = torch.Generator(DEV).manual_seed(seed * 1_000_003 + 17)
    host = np.random.RandomState((seed * 7919 + 13) % (1 << 31))
    s = types.SimpleNamespace(case=case, kind=case["kind"])
    if s.kind == "pages":
        old, new = _lengths(case)
        page = case["page"]
        used = -(-old // page)
        total = int((-(-(old + new) // page)).sum()) + 16
        order = host.permutation(total)
        s.width = int((-(-(old + new) // page)).max()) + 2
        table = np.full((len(old), s.width), -1)
        at = 0
        for b, n in enumerate(used):
            table[b, :n] = order[at:at + n]
            at += n
        s.free_host = np.concatenate([order[at:], np.zeros(at, int)])
        s.count_host, s.table_host, s.old, s.new_host, s.pages = total - at, table, old, new, total
        s.rows, s.longest = int(new.sum()), int((old + new).max())
        s.table, s.lengths, s.new = _int32(table), _int32(old), _int32(new)
        s.keep, s.free, s.count = s.lengths.clone(), _int32(s.free_host), _int32([s.count_host])
        return s
    if s.kind == "store":
        rows, heads, dim, page = case["rows"], case["kv_heads"], case["dim"], case["page"]
        s.pages = -(-rows // page) + 3
        used = host.permutation(s.pages)[:-(-rows // page)]
        s.slots_host = (used[np.arange(rows) // page] * page + np.arange(rows) % page).astype(np.int64)
        if rows > 8:
            s.slots_host[-2:] = -1  # a padded batch's rows
        s.slots = torch.tensor(s.slots_host, device=DEV)
        dtype = DTYPES[case["dtype"]]
        # as an attention layer hands them over: heads before tokens
        s.key = _keys((rows, heads, dim), g).transpose(0, 1).contiguous().to(dtype).transpose(0, 1)
        s.value = _normal((rows, heads, dim), g).transpose(0, 1).contiguous().to(dtype).transpose(0, 1)
        return s
    if s.kind == "attend":
        old, new = _lengths(case)
        heads, dim, page = case["kv_heads"], case["dim"], case["page"]
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
            slots = torch.tensor(s.table_host[b, tokens // page] * page + tokens % page, device=DEV)
            _write(s.store, slots, _keys((len(tokens), heads, dim), g), _normal((len(tokens), heads, dim), g), page)
        s.cu_host = np.concatenate([[0], np.cumsum(new)])
        s.rows, s.longest, s.most = int(new.sum()), int(s.totals.max()), int(new.max())
        s.query = _normal((s.rows, heads * case["groups"], dim), g, 1.5).to(DTYPES[case["dtype"]])
        s.table, s.lengths, s.cu = _int32(s.table_host), _int32(s.totals), _int32(s.cu_host)
        s.scaling = dim ** -0.5
        return s
    rows, vocab = case["rows"], case["vocab"]
    length, prompt = _history(case)
    s.logits = _normal((rows, vocab), g, 3.0).to(DTYPES[case["dtype"]])
    # token frequencies fall off as they do in text
    words = np.minimum((vocab * host.power(0.35, (rows, max(1, case["history"])))).astype(np.int64), vocab - 1)
    s.tokens, s.length, s.prompt = torch.tensor(words, device=DEV), _int32(length), _int32(prompt)
    s.repetition = torch.tensor(host.choice([1.0, 1.05, 1.1, 1.3, 0.9], rows), dtype=torch.float32, device=DEV)
    s.presence = torch.tensor(host.choice([0.0, 0.25, 1.0, -0.5], rows), dtype=torch.float32, device=DEV)
    s.frequency = torch.tensor(host.choice([0.0, 0.125, 0.75], rows), dtype=torch.float32, device=DEV)
    s.bias_ids = s.bias_values = s.bias_cu = s.allowed = s.allowed_row = None
    if case["biased"]:
        count = host.randint(0, case["biased"] + 1, rows)
        count[0] = case["biased"]
        total = int(count.sum())
        s.bias_cu = _int32(np.concatenate([[0], np.cumsum(count)]))
        s.bias_ids = _int32(host.randint(0, vocab, total))
        s.bias_values = torch.tensor(host.choice([-100.0, -2.5, 1.5, 5.0], total), dtype=torch.float32, device=DEV)
    if case["masked"]:
        masks = max(1, rows // 2)
        density = torch.rand(masks, 1, generator=g, device=DEV) ** 2
        bits = torch.rand(masks, -(-vocab // 32) * 32, generator=g, device=DEV) < density
        shifts = torch.arange(32, device=DEV)
        word = (bits.view(masks, -1, 32).long() << shifts).sum(-1)
        s.allowed = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
        s.allowed_row = _int32([r // 2 if r % 2 == 0 and r // 2 < masks else -1 for r in range(rows)])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    kind = s.kind
    if kind == "store":
        s.store = _empty_pages(s.pages, case["kv_heads"], case["page"], case["dim"])
    if not own:
        return s
    for p in (ROOT, os.path.join(ROOT, "dimmer-kv_amd")):
        if p not in sys.path:
            sys.path.insert(0, p)
    import paged_cache
    import reply_controls

    if kind == "pages":
        s.cache = paged_cache.PagedCache(0, 1, 64, s.pages, page=case["page"], requests=case["requests"],
                                         table_pages=s.width, device=DEV)
        for name, value in (("table", s.table), ("lengths", s.lengths), ("free", s.free), ("free_count", s.count)):
            getattr(s.cache, name).copy_(value)
    elif kind in ("store", "attend"):
        s.cache = paged_cache.PagedCache(1, case["kv_heads"], case["dim"], s.pages, page=case["page"],
                                         requests=case.get("requests", 1),
                                         table_pages=s.table.shape[1] if kind == "attend" else s.pages, device=DEV)
        for name in s.store:
            getattr(s.cache, name)[0].copy_(s.store[name][:s.pages])
        del s.store
        if kind == "attend":
            s.cache.table.copy_(s.table)
            s.cache.lengths.copy_(s.lengths)
            s.step = paged_cache.Step(slots=None, positions=None, cu=s.cu, rows=s.rows, longest=s.longest, most=s.most)
        else:
            s.step = paged_cache.Step(slots=s.slots, positions=None, cu=None, rows=case["rows"], longest=0, most=0)
    else:
        s.controls = reply_controls.ReplyControls(
            case["rows"], case["vocab"], repetition=s.repetition, presence=s.presence, frequency=s.frequency,
            bias=None if s.bias_cu is None else (s.bias_ids, s.bias_values, s.bias_cu),
            allowed=None if s.allowed is None else (s.allowed, s.allowed_row), device=DEV)
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    return {"pages": _run_pages, "store": _run_store, "attend": _run_attend, "logits": _run_logits}[s.kind](s)


def _run_pages(s):
    """The new tokens' pages and slots, and the requests cut back to what they were (a draft refused)."""
    if own:
        step = s.cache.assign(s.new, s.rows, longest=s.longest)
        s.cache.trim(s.keep)
        return [step.slots, step.positions, step.cu, s.cache.table, s.cache.lengths, s.cache.free, s.cache.free_count]
    page = s.case["page"]
    old, new = s.lengths.long(), s.new.long().clamp(min=0)
    before, after = (old + page - 1) // page, (old + new + page - 1) // page
    need = after - before
    first = torch.cumsum(need, 0) - need
    column = torch.arange(s.width, device=DEV)
    fresh = (column >= before[:, None]) & (column < after[:, None])
    take = s.count.long() - 1 - (first[:, None] + column - before[:, None])
    table = torch.where(fresh, s.free[take.clamp(0, s.pages - 1)], s.table)
    cu = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0))
    owner = torch.repeat_interleave(torch.arange(old.numel(), device=DEV), new, output_size=s.rows)
    positions = torch.arange(s.rows, device=DEV) - cu[owner] + old[owner]
    slots = table[owner, positions // page].long() * page + positions % page
    # back to the kept lengths: the pages return to the places they came from
    keep = torch.minimum(old + new, s.keep.long().clamp(min=0))
    left = (keep + page - 1) // page
    given = after - left
    ahead = torch.cumsum(given, 0) - given
    count = s.count.long() - need.sum()
    gone = (column >= left[:, None]) & (column < after[:, None])
    back = count + given.sum() - 1 - (ahead[:, None] + column - left[:, None])
    free = torch.cat([s.free, s.free[:1]])
    free[torch.where(gone, back, torch.full_like(back, s.pages)).flatten()] = table.flatten()
    table = torch.where(gone, torch.full_like(table, -1), table)
    return [slots, positions, cu.int(), table, keep.int(), free[:-1], (count + given.sum()).int()]


def _run_store(s):
    """Keys and values of a step into the cache, and the same rows out of it."""
    if own:
        s.cache.store(0, s.key, s.value, s.step)
        return list(s.cache.load(0, s.slots, dtype=s.key.dtype))
    page, heads, dim = s.case["page"], s.case["kv_heads"], s.case["dim"]
    _write(s.store, s.slots, s.key, s.value, page)
    key, value = _rows(s.store, s.slots, heads, page, dim)
    return [key.to(s.key.dtype), value.to(s.value.dtype)]


def _run_attend(s):
    case = s.case
    window = case["window"]
    if own:
        return s.cache.attend_rows(0, s.query, s.step, scaling=s.scaling, window=window or None)
    page, heads, dim, groups = case["page"], case["kv_heads"], case["dim"], case["groups"]
    out = torch.empty_like(s.query)
    for b, (total, new) in enumerate(zip(s.totals.tolist(), s.new_host.tolist())):
        at = torch.arange(total, device=DEV)
        key, value = _rows(s.store, s.table[b].long()[at // page] * page + at % page, heads, page, dim)
        begin = int(s.cu_host[b])
        query = s.query[begin:begin + new].float().unflatten(1, (heads, groups))
        place = torch.arange(total - new, total, device=DEV)
        hidden = at[None] > place[:, None]
        if window:
            hidden |= at[None] <= place[:, None] - window
        for h in range(heads):
            scores = torch.matmul(query[:, h].reshape(new * groups, dim), key[:, h].t().contiguous()) * s.scaling
            scores = scores.view(new, groups, total).masked_fill(hidden[:, None], float("-inf"))
            scores = torch.exp(scores - scores.amax(-1, keepdim=True))
            mixed = torch.matmul(scores.view(new * groups, total), value[:, h]).view(new, groups, dim)
            out[begin:begin + new, h * groups:(h + 1) * groups] = (mixed / scores.sum(-1, keepdim=True)).to(out.dtype)
    return out


def _run_logits(s):
    """The adjusted logits and each row's pick."""
    if own:
        return list(s.controls.apply(s.logits, s.tokens, s.length, s.prompt))
    rows, vocab = s.logits.shape
    x = s.logits.float()
    at = torch.arange(s.tokens.shape[1], device=DEV)[None]
    held = (at < s.length[:, None]) & (s.tokens >= 0) & (s.tokens < vocab)
    reply = held & (at >= s.prompt[:, None])
    place = s.tokens.clamp(0, vocab - 1)
    seen = torch.zeros(rows, vocab, dtype=torch.int32, device=DEV).scatter_add_(1, place, held.int())
    count = torch.zeros(rows, vocab, dtype=torch.int32, device=DEV).scatter_add_(1, place, reply.int())
    rate = s.repetition[:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rate, x * rate), x)
    less = s.frequency[:, None] * count.float() + s.presence[:, None]
    x = torch.where(count > 0, x - less, x)
    if s.bias_cu is not None:
        amount = (s.bias_cu[1:] - s.bias_cu[:-1]).long()
        row = torch.repeat_interleave(torch.arange(rows, device=DEV), amount, output_size=s.bias_ids.numel())
        # an id listed twice takes its last value
        last = torch.full((rows * vocab,), -1, dtype=torch.int64, device=DEV)
        last.scatter_reduce_(0, row * vocab + s.bias_ids, torch.arange(row.numel(), device=DEV), "amax")
        last = last.view(rows, vocab)
        x = torch.where(last >= 0, x + s.bias_values[last.clamp(min=0)], x)
    if s.allowed is not None:
        bits = ((s.allowed[:, :, None] >> torch.arange(32, device=DEV)) & 1).flatten(1)[:, :vocab].bool()
        free = (s.allowed_row < 0)[:, None]
        x = torch.where(free | bits[s.allowed_row.clamp(min=0).long()], x, torch.full_like(x, float("-inf")))
    best = x.amax(-1, keepdim=True)
    index = torch.arange(vocab, device=DEV)
    pick = torch.where(x == best, index, vocab).amin(-1)
    pick = torch.where(best[:, 0] == float("-inf"), torch.full_like(pick, -1), pick)
    return [x.to(s.logits.dtype), pick]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "pages":
        old, new = _lengths(case)
        page = case["page"]
        moved = int((-(-(old + new) // page) - -(-old // page)).sum())
        # lengths and new tokens, lengths out, cumulative counts; slots and positions; a page: read, into the table,
        # out of it and back
        return {"bytes": 16 * len(old) + 16 * int(new.sum()) + 16 * moved, "flops": 4 * int(new.sum())}
    if kind == "store":
        element = torch.finfo(DTYPES[case["dtype"]]).bits // 8
        values = 2 * case["rows"] * case["kv_heads"] * case["dim"]
        # in, the codes written and read, out
        return {"bytes": int(values * (2 * element + 2 * (0.5 + 1 / 32))) + 16 * case["rows"], "flops": 6 * values}
    if kind == "attend":
        old, new = _lengths(case)
        heads, dim, groups, window = case["kv_heads"], case["dim"], case["groups"], case["window"]
        element = torch.finfo(DTYPES[case["dtype"]]).bits // 8
        seen = pairs = 0
        for o, n in zip(old.tolist(), new.tolist()):
            first = 0 if not window else max(0, o + 1 - window)
            seen += o + n - first
            place = np.arange(o + 1, o + n + 1, dtype=np.int64)
            pairs += int(np.minimum(place, window).sum() if window else place.sum())
        rows = int(new.sum())
        return {"bytes": int(2 * seen * heads * dim * (0.5 + 1 / 32)) + 2 * rows * heads * groups * dim * element,
                "flops": 4 * pairs * heads * groups * dim}
    rows, vocab = case["rows"], case["vocab"]
    element = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    length, _ = _history(case)
    masks = max(1, rows // 2) * -(-vocab // 32) * 4 if case["masked"] else 0
    return {"bytes": 2 * rows * vocab * element + 8 * int(length.sum()) + masks + 8 * rows * case["biased"],
            "flops": 4 * rows * vocab}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    return {"pages": _exact_pages, "store": _exact_store, "attend": _exact_attend, "logits": _exact_logits}[s.kind](s)


def _exact_pages(s):
    """Request by request: pages off the stack one at a time, and back on it in the opposite order."""
    page = s.case["page"]
    table, stack = s.table_host.copy(), s.free_host.copy()
    top = s.count_host
    slots, positions, taken = [], [], []
    for b, (old, new) in enumerate(zip(s.old.tolist(), s.new_host.tolist())):
        for at in range(-(-old // page), -(-(old + new) // page)):
            top -= 1
            table[b, at] = stack[top]
            taken.append((b, at))
        place = np.arange(old, old + new)
        positions.append(place)
        slots.append(table[b, place // page] * page + place % page)
    for b, at in reversed(taken):
        stack[top] = table[b, at]
        table[b, at] = -1
        top += 1
    cu = np.concatenate([[0], np.cumsum(s.new_host)])
    whole = lambda a, t: torch.tensor(np.asarray(a), dtype=t, device=DEV)
    return [whole(np.concatenate(slots), torch.int64), whole(np.concatenate(positions), torch.int64),
            whole(cu, torch.int32), whole(table, torch.int32), whole(s.old, torch.int32), whole(stack, torch.int32),
            whole([top], torch.int32)]


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


def _exact_store(s):
    gone = (s.slots < 0)[:, None, None]
    return [_nearest(s.key).masked_fill(gone, 0.0), _nearest(s.value).masked_fill(gone, 0.0)]


def _unpacked(s, b, head):
    """float64 keys and values [total, D] of one request's head, byte by byte of its pages."""
    page, heads, dim = s.case["page"], s.case["kv_heads"], s.case["dim"]
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


def _exact_attend(s):
    case = s.case
    heads, groups, window = case["kv_heads"], case["groups"], case["window"]
    out = torch.zeros(s.query.shape, dtype=torch.float64, device=DEV)
    for b in range(case["requests"]):
        total, begin, end = int(s.totals[b]), int(s.cu_host[b]), int(s.cu_host[b + 1])
        at = torch.arange(total, device=DEV)
        for h in range(heads):
            key, value = _unpacked(s, b, h)
            for g in range(h * groups, (h + 1) * groups):
                for lo in range(begin, end, 1024):
                    hi = min(end, lo + 1024)
                    place = torch.arange(total - (end - lo), total - (end - hi), device=DEV)[:, None]
                    visible = at[None] <= place
                    if window:
                        visible &= at[None] > place - window
                    logit = s.query[lo:hi, g].double() @ key.t().contiguous() * s.scaling
                    weight = torch.softmax(torch.where(visible, logit, torch.full_like(logit, -math.inf)), -1)
                    out[lo:hi, g] = weight @ value
    return out


def _exact_logits(s):
    rows, vocab = s.logits.shape
    out = torch.empty(rows, vocab, dtype=torch.float64, device=DEV)
    pick = []
    length, prompt = s.length.tolist(), s.prompt.tolist()
    for r in range(rows):
        x = s.logits[r].double()
        history, reply = s.tokens[r, :length[r]], s.tokens[r, prompt[r]:length[r]]
        known = history[(history >= 0) & (history < vocab)].unique()
        rate = s.repetition[r].double()
        x[known] = torch.where(x[known] > 0, x[known] / rate, x[known] * rate)
        ids, count = reply[(reply >= 0) & (reply < vocab)].unique(return_counts=True)
        x[ids] -= s.frequency[r].double() * count + s.presence[r].double()
        if s.bias_cu is not None:
            lo, hi = int(s.bias_cu[r]), int(s.bias_cu[r + 1])
            wanted = dict(zip(s.bias_ids[lo:hi].tolist(), s.bias_values[lo:hi].tolist()))
            if wanted:
                at = torch.tensor(list(wanted), device=DEV)
                x[at] += torch.tensor(list(wanted.values()), dtype=torch.float64, device=DEV)
        if s.allowed is not None and int(s.allowed_row[r]) >= 0:
            words = s.allowed[int(s.allowed_row[r])].cpu().numpy().view(np.uint32)
            bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:vocab]
            x[torch.tensor(bits == 0, device=DEV)] = -math.inf
        out[r] = x
        value, at = x.max(0)
        pick.append(-1 if float(value) == -math.inf else int((x == value).nonzero()[0]))
    return [out, torch.tensor(pick, dtype=torch.int64, device=DEV)]
