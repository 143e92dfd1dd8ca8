"""Distillation on the CPU at low temperatures."""

import pytest
import torch

import exact_logits
from alignment_reference import near
from test1_amd.distillation import linear_distill


@pytest.mark.parametrize("temperature", [1.0, 0.01, 1e-4, 1e-9, 1e-20, 1e-30])
@pytest.mark.parametrize("kind,rest", [("forward", True), ("forward", False), ("reverse", True)])
def test_low_temperatures(kind, rest, temperature):
    for dtype in (torch.float32, torch.bfloat16):
        hidden, weight, ids, logps, mask, up = exact_logits.inputs((12, 64, 300, 20), dtype, "cpu")
        up = up * temperature
        want, bound = exact_logits.distill(hidden, weight, ids, logps, mask, temperature, kind, rest, up)
        hr, wr = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        loss = linear_distill(hr, wr, ids, logps, mask, temperature, kind, rest)
        for got, w, b in zip((loss.detach(), *torch.autograd.grad(loss, (hr, wr), up)), want, bound):
            near(got, w, b)
