"""Recorded calls, contexts and places of shaped scores, on the CPU."""

from __future__ import annotations

import pytest
import torch

import dkv_hip


def test_every_recorded_input_refuses_its_gradient():
    first, second, plain = torch.zeros(3, requires_grad=True), torch.zeros(3, requires_grad=True), torch.zeros(3)
    out = dkv_hip._recorded("this", torch.ones(3), first, None, plain, second)
    for t in (first, second):
        with pytest.raises(RuntimeError, match="this has no backward pass"):
            torch.autograd.grad(out.sum(), t, allow_unused=True, retain_graph=True)
    assert dkv_hip._recorded("this", plain, plain, None) is plain
    with torch.no_grad():
        assert not dkv_hip._recorded("this", torch.ones(3), first).requires_grad
