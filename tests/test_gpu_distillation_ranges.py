"""Distillation on the GPU at low temperatures, where logits over the temperature
leave what exponentials and even whole numbers of fp32 hold."""

import pytest
import torch

import exact_logits
from alignment_reference import near
from test1_amd.distillation import linear_distill

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
# in tiles of small products, of odd rows that the tiles do not take, in pieces, with rows of D that are close
SHAPES = [(70, 64, 700, 20), (70, 40, 300, 6), (300, 128, 3000, 40), (400, 2048, 50_000, 9)]


def check(shape, dtype, dev, temperature, kind, rest):
    hidden, weight, ids, logps, mask, up = exact_logits.inputs(shape, dtype, dev)
    up = up * temperature   # derivatives by the logits over the temperature
    want, bound = exact_logits.distill(hidden, weight, ids, logps, mask, temperature, kind, rest, up)
    with torch.no_grad():
        near(linear_distill(hidden, weight, ids, logps, mask, temperature, kind, rest), want[0], bound[0])
    hr, wr = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    loss = linear_distill(hr, wr, ids, logps, mask, temperature, kind, rest)
    for got, w, b in zip((loss.detach(), *torch.autograd.grad(loss, (hr, wr), up, retain_graph=True)), want, bound):
        near(got, w, b)
    for got, w, b in zip(torch.autograd.grad(loss, (hr, wr), up), want[1:], bound[1:]):   # made again
        near(got, w, b)


@pytest.mark.parametrize("temperature", [1.0, 0.01, 1e-4, 1e-6, 1e-8, 1e-9, 1e-12, 1e-20, 1e-30])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind,rest", [("forward", False), ("reverse", True)])
def test_low_temperatures(dev, shape, temperature, kind, rest):
    for dtype in TYPES if shape[1] < 2048 else TYPES[:1]:
        check(shape, dtype, dev, temperature, kind, rest)
