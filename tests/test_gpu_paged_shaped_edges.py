"""Shaped scores where one row or input could spoil another's."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged_attend import DEV, TYPES, build
from test_gpu_paged_shaped import compare, numbers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["", "slopes", "sinks+first"])
@pytest.mark.parametrize("old,new,dim", [(59, 1, 64), (300, 40, 64), (300, 40, 128), (130, 3, 256)])
@pytest.mark.parametrize("dtype,cap", [(dtype, cap) for dtype in ("f32", "f16", "bf16") for cap in (200.0, 1e4, 1e5)] +
                         [("f32", 1e6), ("bf16", 1e6)])
def test_caps_beside_rows_that_reach_them(dtype, cap, old, new, dim, kind):
    """Heads whose scores pass four fifths of the cap, up and down, in the tiles of heads whose scores are about 1.  The bound
    is compare's: a row whose own scores stay within half of its cap is off by the size of those and not of the cap, for
    caps above 128 whatever the type.  (The far heads' scores at ten tokens are z = 0.8 cap, of some 0.1 cap at the others.)"""
    print(f"[case] caps beside {kind} {old}+{new} dim={dim} cap={cap} {dtype}", flush=True)
    cache, step = build([old], [new], 1, dim, 16, seed=3)
    keys = cache.load(0, cache.slots(0, 0, old + new), torch.float32)[0][:, 0]
    g = torch.Generator(DEV).manual_seed(1)
    query = torch.randn(new, 4, dim, generator=g, device=DEV) * (0.8 / dim ** 0.5)
    ten = torch.arange(10, device=DEV) * (old // 10) + 3
    near = keys[ten].double().cpu()  # the shortest vector of these ten scores
    far = (near.T @ torch.linalg.solve(near @ near.T, torch.full((10,), 0.8 * cap, dtype=torch.float64))).float().to(DEV)
    query[:, 0], query[:, 2] = far, -far
    query = query.to(TYPES[dtype])
    assert query.isfinite().all()
    z = query.double() @ keys.double().T
    assert (z[:, [0, 2]].abs().amax(-1) > 0.7 * cap).all() and (z[:, [1, 3]].abs() < 6.0).all()
    made = dict(cap=cap)
    if "slopes" in kind:
        made["slopes"] = torch.tensor([0.5, 0.01, 0.002, 0.0], device=DEV)
    if "sinks" in kind:
        made["sinks"], made["first"] = numbers(4, 5), (step.positions - 250).clamp(min=0)
    got = cache.attend_rows(0, query, step, scaling=1.0, **made)
    compare(cache, step, query, got, scaling=1.0, **made)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,old,new", [(64, 1, 59, 1), (128, 1, 9000, 2), (64, 2, 20000, 1), (64, 1, 300, 45), (256, 1, 300, 45),
                                               (64, 8, 0, 2100), (64, 16, 0, 6600)])
def test_sinks_past_all_scores(dim, heads, old, new, dtype):
    """A sink of +infinity, or one that is finite and past all scores by any amount, takes all: rows are 0, as
    sum e^z v / (sum e^z + e^s) is; a sink that is no number makes its rows NaN; other heads' are as without."""
    print(f"[case] sinks past all {old}+{new} dim={dim} heads={heads} {dtype}", flush=True)
    cache, step = build([old], [new], heads, dim, 64)
    query = torch.randn(new, 5 * heads, dim, generator=torch.Generator(DEV).manual_seed(2), device=DEV).to(TYPES[dtype])
    first = torch.zeros_like(step.positions)
    mild = torch.tensor([-1.0, -1.0, -1.0, -1.0, 0.5], device=DEV).repeat(heads)
    for large in ((float("inf"), 3.4e38, 2.5e38), (1e4, 7.77e8, 3.3e12), (1.23e17, 5.4e29, 2.3e38)):
        sinks = torch.tensor([*large, float("nan"), 0.5], device=DEV).repeat(heads)
        for made in (dict(), dict(cap=5.0), dict(first=first), dict(slopes=torch.full_like(sinks, 0.1))):
            got = cache.attend_rows(0, query, step, sinks=sinks, **made).unflatten(1, (heads, 5))
            want = cache.attend_rows(0, query, step, sinks=mild, **made).unflatten(1, (heads, 5))
            assert not got[:, :, :3].any() and got[:, :, 3].isnan().all() and torch.equal(got[:, :, 4], want[:, :, 4])


def test_every_recorded_input_refuses_its_gradient():
    cache, step = build([50, 9], [2, 3], 2, 64, 16)
    given = [torch.randn(5, 6, 64, device=DEV), numbers(6, 1), numbers(6, 2).abs()]
    for t in given:
        t.requires_grad_()
    got = cache.attend_rows(0, given[0], step, sinks=given[1], slopes=given[2])
    for t in given:
        with pytest.raises(RuntimeError, match="no backward pass"):
            torch.autograd.grad(got.sum(), t, allow_unused=True, retain_graph=True)
