"""Rotated appends where two roundings, or a bound on an exact value, would show."""

from __future__ import annotations

from fractions import Fraction

import pytest
import torch

from test_gpu_paged_append import inputs, make, tables
from test_gpu_paged_attend import DEV, TYPES

pytestmark = pytest.mark.gpu
CODES = [Fraction(x) for x in ("0", "0.5", "1", "1.5", "2", "3", "4", "6")]
BITS = {"f32": 24, "f16": 11, "bf16": 8}


def nearest(x: Fraction, bits: int) -> float:
    """x, of the type's normal range, rounded to ``bits`` bits, ties to the even one."""
    if x == 0:
        return 0.0
    unit = Fraction(1)
    while abs(x) / unit >= 1 << bits:
        unit *= 2
    while abs(x) / unit < 1 << (bits - 1):
        unit /= 2
    return float(round(x / unit) * unit)  # (round of a fraction is to the even one)


def nearest_code(x: Fraction) -> float:
    """x to the nearest of the 4-bit values of exponent 0, ties to the even code."""
    size = min(abs(x), Fraction(6))
    place = min(range(8), key=lambda i: (abs(CODES[i] - size), i % 2))
    return float(CODES[place]) * (-1 if x < 0 else 1)


def turned(row, cos, sin, interleaved):
    """The exact rotation of one row [dim] of finite floats by one row of tables."""
    row, pairs = [Fraction(float(x)) for x in row], len(cos)
    out = list(row)
    for i in range(pairs):
        one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        c, s = Fraction(float(cos[i])), Fraction(float(sin[i]))
        out[one], out[two] = row[one] * c - row[two] * s, row[two] * c + row[one] * s
    return out


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (128, 32)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_keys_whose_sums_pass_64_bits(dtype, dim, rotary, interleaved):
    """Keys on the border of two codes, or of two exponents, that the other product of the sum takes past it by 2^-60 of
    them, up or down: the code is the exact value's nearest."""
    cache, step = make([32], 1, dim)
    pairs = rotary // 2
    one, two = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, pairs), slice(pairs, rotary))
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -1.25, -2.5, -5.0])
    little = 2.0 ** -24  # a value of every type
    key = torch.zeros(32, 1, dim)
    key[:, 0, one] = ties[torch.arange(32 * pairs).reshape(32, pairs) % 11]
    key[:, 0, two] = torch.tensor([little, -little])[torch.arange(32) % 2, None]
    key[:, 0, one][:, ::8] = 6.0  # the largest of each block: exponent 0, or, next to its border, whichever is exact
    key[::4, 0, one] = key[::4, 0, one].clamp(max=5.0)
    key[::4, 0, one][..., ::8] = 7.0
    key = key.to(TYPES[dtype]).to(DEV)
    for c, s in ((1.0, 2.0 ** -36), (1.0, -(2.0 ** -36)), (1.0, 2.0 ** -50)):
        cos, sin = torch.full((32, pairs), c, device=DEV), torch.full((32, pairs), s, device=DEV)
        cache.append(0, None, key, key, step, cos, sin, interleaved=interleaved)
        held = cache.load(0, step.slots, torch.float32)[0].double().cpu().numpy()
        for t in range(32):
            exact = turned(key[t, 0].tolist(), cos[t].tolist(), sin[t].tolist(), interleaved)
            for at in range(0, dim, 32):
                block = exact[at:at + 32]
                scale = 2 if max(abs(x) for x in block) >= 7 else 1
                if max(abs(x) for x in block) < Fraction(7, 2):
                    continue  # a block of smaller exponents: rows of test_rotations_next_to_a_border
                want = [nearest_code(x / scale) * scale for x in block]
                assert want == held[t, 0, at:at + 32].tolist(), (t, at, c, s)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_queries_whose_sums_pass_64_bits(interleaved, dtype):
    """x cos on the middle of two numbers of the type, y sin 2^-60 of it: the result is the exact value's nearest.  Beside
    random rows, which are rounded once too."""
    cache, step = make([16], 1, 64)
    bits = BITS[dtype]
    query = torch.randn(16, 1, 64, generator=torch.Generator().manual_seed(4))
    one, two = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    angles = torch.rand(16, 32, generator=torch.Generator().manual_seed(5)) * 6.0
    cos, sin = angles.cos(), angles.sin()
    little = 2.0 ** -24
    # products of 1 + 2^-k and 1 + 2^-k' whose last bit is half of the type's last
    x, c = (1.0 + 2.0 ** -12, 1.0 + 2.0 ** -12) if bits == 24 else (1.0, 1.0 + 2.0 ** -bits)
    query[:8, 0, one], query[:8, 0, two] = x, torch.tensor([little, -little])[torch.arange(8) % 2, None]
    cos[:8], sin[:8] = c, torch.tensor([2.0 ** -36, 2.0 ** -36, -(2.0 ** -36), 0.0]).repeat(2)[:, None]
    query = query.to(TYPES[dtype])
    got = cache.append(0, query.to(DEV), query.to(DEV), query.to(DEV), step, cos.to(DEV), sin.to(DEV), interleaved=interleaved)
    positions = step.positions.tolist()
    for t in range(16):
        exact = turned(query[t, 0].tolist(), cos[positions[t]].tolist(), sin[positions[t]].tolist(), interleaved)
        large = [i for i, v in enumerate(exact) if abs(v) > 2.0 ** -13]  # (smaller ones may be subnormal float16)
        assert len(large) >= 32
        have = got[t, 0].double().tolist()
        assert [nearest(exact[i], bits) for i in large] == [have[i] for i in large], t


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 32), (64, 48), (128, 32), (128, 64), (128, 96), (256, 16), (256, 64), (256, 192)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_dimensions_that_stay(dtype, dim, rotary, interleaved):
    """Blocks of dimensions behind the rotated ones hold the bytes that store writes, the sign of zeros and values on the
    border of two codes among them; the queries' dimensions there keep their bits."""
    cache, step = make([40], 2, dim)
    query, key, value = inputs(40, 4, 2, dim, dtype, 3)
    ties = torch.tensor([0.0, -0.0, 0.25, -0.25, 0.75, 1.25, -1.75, 2.5, 3.5, -5.0, 6.0], device=DEV)
    for t in (query, key):
        t[::2, :, rotary:] = ties[torch.arange(t[::2, :, rotary:].numel(), device=DEV) % 11].view_as(t[::2, :, rotary:]).to(t.dtype)
        t[5] = -0.0
    cos, sin = tables(40, rotary // 2)
    got = cache.append(0, query, key, value, step, cos, sin, interleaved=interleaved)
    bits = {2: torch.int16, 4: torch.int32}[query.element_size()]
    assert torch.equal(got[..., rotary:].contiguous().view(bits), query[..., rotary:].contiguous().view(bits))
    keys = cache.load(0, step.slots, torch.float32)[0]
    codes, scales = cache.key_codes.clone(), cache.key_scales.clone()
    cache.store(0, key, value, step)
    stored = cache.load(0, step.slots, torch.float32)[0]
    whole = -(-rotary // 32) * 32  # the first block that nothing of is rotated
    if whole < dim:
        assert torch.equal(keys[..., whole:].contiguous().view(torch.int32), stored[..., whole:].contiguous().view(torch.int32))
        page = cache.page
        for a, b, width, at in ((codes, cache.key_codes, dim // 2, whole // 2), (scales, cache.key_scales, dim // 32, whole // 32)):
            a, b = (t[0].view(-1, 2, page, width)[..., at:] for t in (a, b))
            assert torch.equal(a, b)
    if rotary % 32:  # a block of both: a zero keeps its sign whatever the block's exponent
        part = key[..., rotary:whole].float()
        zero = part == 0
        assert zero.any() and torch.equal(keys[..., rotary:whole][zero].signbit(), part[zero].signbit())


@pytest.mark.parametrize("x,y,want", [(float("inf"), 3e38, (float("inf"), float("inf"))),
                                      (3e38, -float("inf"), (float("inf"), -float("inf")))])
def test_infinities_beside_products_past_float32(x, y, want):
    """An infinite query beside a finite product that float32 does not hold is infinite, not NaN: x - 1.5 y, y + 1.5 x."""
    cache, step = make([4], 1, 64)
    query = torch.ones(4, 1, 64, device=DEV).bfloat16()
    query[1, 0, 3], query[1, 0, 35] = x, y
    cos, sin = torch.ones(4, 32, device=DEV), torch.full((4, 32), 1.5, device=DEV)
    got = cache.append(0, query, query, query, step, cos, sin).float()
    assert (got[1, 0, 3].item(), got[1, 0, 35].item()) == want
    assert got.isinf().sum() == 2 and not got.isnan().any()


def test_layers_beside_the_one_that_is_written():
    """Appends to a layer leave the codes and exponents of the others as they are, whatever they held."""
    cache, step = make([300, 41], 4, 64, page=64, layers=3)
    query, key, value = inputs(step.rows, 8, 4, 64, "f16")
    cos, sin = tables(300, 32)
    names = ("key_codes", "key_scales", "value_codes", "value_scales")
    for name in names:
        t = getattr(cache, name)
        t.copy_(torch.randint(0, 255, t.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(1)))
    before = {name: getattr(cache, name).clone() for name in names}
    cache.append(1, query, key, value, step, cos, sin)
    for name in names:
        held = getattr(cache, name)
        assert torch.equal(held[0], before[name][0]) and torch.equal(held[2], before[name][2])
        assert not torch.equal(held[1], before[name][1])


def test_every_recorded_input_refuses_its_gradient():
    cache, step = make([5], 2, 64)
    query, key, value = inputs(5, 4, 2, 64, "f32")
    cos, sin = tables(8, 32)
    for t in (query, cos, sin):
        t.requires_grad_()
    got = cache.append(0, query, key, value, step, cos, sin)
    for t in (query, cos, sin):
        with pytest.raises(RuntimeError, match="no backward pass"):
            torch.autograd.grad(got.sum(), t, allow_unused=True, retain_graph=True)
