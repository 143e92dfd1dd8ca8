"""Distillation on the GPU at low temperatures, where logits over the temperature
leave what exponentials and even whole numbers of fp32 hold."""

import pytest
import torch

import exact_logits
from alignment_reference import near
from distill_reference import distill
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
@pytest.mark.parametrize("kind,rest", [("forward", False), ("reverse", True), ("forward", True)])
def test_low_temperatures(dev, shape, temperature, kind, rest):
    for dtype in TYPES if shape[1] < 2048 else TYPES[:1]:
        check(shape, dtype, dev, temperature, kind, rest)


# tokens, hidden, vocabulary, words, masked: few tokens; a product of the framework's own; one of close rows
@pytest.mark.parametrize("shape", [(70, 64, 257, 1, False), (70, 64, 300, 44, False), (300, 128, 895, 127, True), (4200, 2048, 513, 1, False),
                                   (4200, 2048, 4097, 1, True)])
def test_a_last_span_whose_words_are_all_named(dev, shape):
    """What pads the vocabulary to a whole span stays out of the hidden gradient, where all other words are far
    below: there is no word of the last span that the padding could be relative to."""
    n, h, v, k, masked = shape
    for dtype in (torch.bfloat16, torch.float16):
        for below in (2, 4):
            g = torch.Generator(device=dev).manual_seed(v + below)
            hidden = torch.randint(0, 3, (n, h), generator=g, device=dev).to(dtype)
            hidden[:, 64:] = 0   # logits of the others around -128 and -256
            weight = torch.randint(-1, 2, (v, h), generator=g, device=dev)
            weight[:v // 256 * 256] -= below
            weight = weight.to(dtype)
            ids = torch.arange(v - k, v, device=dev).expand(n, k).contiguous()
            logps = torch.log_softmax(torch.randn(n, k + 1, generator=g, device=dev), dim=1)[:, :k].contiguous()
            mask = torch.rand(n, generator=g, device=dev) < (0.8 if masked else 2.0)
            up = torch.randn(n, generator=g, device=dev) / n
            want, bound = exact_logits.distill(hidden, weight, ids, logps, mask, 1.0, "forward", True, up)
            hr, wr = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
            loss = linear_distill(hr, wr, ids, logps, mask if masked else None)
            for got, w, b in zip((loss.detach(), *torch.autograd.grad(loss, (hr, wr), up)), want, bound):
                near(got, w, b)


@pytest.mark.parametrize("kind,rest", [("forward", True), ("forward", False), ("reverse", True)])
@pytest.mark.parametrize("gap", [700.0, 1000.0, 5000.0])
def test_a_rest_far_below_the_words(dev, gap, kind, rest):
    """All words outside the teacher's `gap` nats or so below: their mass leaves the exponents of 64 bits, its
    logarithm and the derivative they share do not.  By large hidden states, and by the temperature."""
    n, h, v, k = 70, 64, 700, 5
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        for temperature in (1.0, 0.01):
            g = torch.Generator(device=dev).manual_seed(3)
            hidden = (torch.rand(n, h, generator=g, device=dev) + 0.5) * (gap * temperature / h)
            weight = torch.rand(v, h, generator=g, device=dev) * 0.02 - 1.0
            ids = torch.rand(n, v, generator=g, device=dev).argsort(dim=1)[:, :k].contiguous()
            ids[:] = ids[0]
            weight[ids[0]] += 1.0
            hidden, weight = hidden.to(dtype), weight.to(dtype)
            logps = torch.log_softmax(torch.randn(n, k + 1, generator=g, device=dev), dim=1)[:, :k].contiguous()
            up = torch.randn(n, generator=g, device=dev) * temperature
            want, bound = distill(hidden, weight, ids, logps, None, 1 / temperature, kind, rest, grad=up)
            assert want[0].isfinite().all() and (kind == "reverse" or not rest or (want[0] > 50).any())
            hr, wr = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
            loss = linear_distill(hr, wr, ids, logps, None, temperature, kind, rest)
            for got, w, b in zip((loss.detach(), *torch.autograd.grad(loss, (hr, wr), up)), want, bound):
                near(got, w, b)


@pytest.mark.parametrize("temperature", [30.0, 1e6, 1e30])
@pytest.mark.parametrize("kind,rest", [("forward", False), ("reverse", True), ("forward", True)])
def test_high_temperatures(dev, temperature, kind, rest):
    for shape in SHAPES[:3]:
        for dtype in TYPES:
            check(shape, dtype, dev, temperature, kind, rest)


def test_calls_beside_each_other_and_in_other_modes(dev):
    """Two steps on two streams at once; under inference mode and autocast; of one token, of more dimensions, of none."""
    hidden, weight, ids, logps, mask, up = exact_logits.inputs((700, 512, 30_000, 20), torch.bfloat16, dev)

    def step():
        hr, wr = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        loss = linear_distill(hr, wr, ids, logps, mask, 20.0)
        return loss.detach(), *torch.autograd.grad(loss, (hr, wr), up)

    want = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams * 2:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want))
    with torch.inference_mode():
        assert torch.equal(linear_distill(hidden.clone(), weight, ids, logps, mask, 20.0), want[0])
    with torch.autocast("cuda", dtype=torch.float16):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
    each = linear_distill(hidden, weight, ids, logps, None, 20.0)
    one = linear_distill(hidden[3], weight, ids[3], logps[3], torch.ones((), dtype=torch.bool, device=dev), 20.0)
    # another tile's order of sums: 512 terms in a row of 8 U on each side, and the result's rounding
    assert one.shape == () and (one - each[3]).abs() <= (1040 + 2 * each[3].abs()) * 2.0 ** -24
    cube = linear_distill(hidden.view(7, 10, 10, 512), weight, ids.view(7, 10, 10, 20), logps.view(7, 10, 10, 20), None, 20.0)
    assert torch.equal(cube.flatten(), each)
    hr, wr = hidden[:0].clone().requires_grad_(True), weight.clone().requires_grad_(True)
    loss = linear_distill(hr, wr, ids[:0], logps[:0], mask[:0])
    gh, gw = torch.autograd.grad(loss.sum(), (hr, wr))
    assert loss.shape == (0,) and gh.shape == (0, 512) and (gw == 0).all()
