"""Token log-probabilities of fp16 operands where the type's range ends."""

import pytest
import torch

from alignment_reference import HALF, U, logps, near
from test1_amd import linear_logps as module
from test1_amd.linear_logps import linear_logps
from test_gpu_linear_logps import inputs

pytestmark = pytest.mark.gpu

# kernels of few tokens, of many, a library's products, rows outside the tiles
SHAPES = [(60, 128, 5000), (200, 320, 9000), (300, 896, 1540), (1800, 2560, 5001), (64, 65, 9000), (40, 1024, 50_257)]


def in_chunks(monkeypatch):
    monkeypatch.setattr(module, "_KEEP_BYTES", 0)
    monkeypatch.setattr(module, "_AGAIN_BYTES", 2 * 1024 * 64)
    monkeypatch.setattr(module, "_chunk_rows", lambda vocab: 50)


@pytest.mark.parametrize("chunks", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_the_largest_hidden_states(dev, shape, chunks, monkeypatch):
    """Up to the type's largest number, in the row whose factor is the largest."""
    hidden, weight, labels, up = inputs(shape, torch.float16, dev)
    hidden[3, :4] = 65504.0
    hidden[4, :4] = -40000.0
    weight[:, :4] *= 2.0 ** -13
    labels[3] = 5
    up[3] = 0.99
    if chunks:
        in_chunks(monkeypatch)
    want, bound = logps(hidden, weight, labels, grad=up)
    hidden.requires_grad_(True)
    weight.requires_grad_(True)
    gh, gw = torch.autograd.grad(linear_logps(hidden, weight, labels), (hidden, weight), up)
    assert gh.isfinite().all() and gw.isfinite().all()
    near(gh, want[1], bound[1])
    near(gw, want[2], bound[2])


def exact(hidden, weight, labels, up):
    """(grad_hidden, grad_weight) in 64 bits and the bounds of an evaluation whose
    16-bit operands keep their precision: as ``logps`` counts, but with 2^14
    between an operand's unit and the type's, so that a subnormal is off by 2^-39
    of a row's factor for each of the two roundings, and a weighted hidden row by
    2^-24 of the largest factor times the share of D."""
    h, w = hidden.double(), weight.double()
    rows, at = torch.arange(len(labels), device=h.device), labels.clamp(min=0)
    z = h @ w.t()
    ez = (h.abs() @ w.abs().t()).amax(1) * (2 * h.shape[1] + 2) * U
    lse = torch.logsumexp(z, 1)
    big = z.abs().amax(1) + lse.abs()
    g = torch.where(labels == -100, torch.zeros_like(lse), up.double())
    p = torch.exp(z - lse[:, None])
    dz = -p
    dz[rows, at] = -torch.expm1(z[rows, at] - lse)
    rest = dz[rows, at].clamp(min=2.0 ** -24)
    dz = dz * g[:, None]
    half, tiny = HALF[torch.float16]
    edz = dz.abs() * (2 * half + 8 * U)
    edz += (p * (2 * ez + (512 + 8 * big) * U)[:, None] + 2 * tiny * 2.0 ** -14) * g.abs()[:, None]
    gh, gw = dz @ w, dz.t() @ h
    egh = edz @ w.abs() + (dz.abs() @ w.abs()) * (2 * w.shape[0] * U) + half * gh.abs() + tiny
    egw = edz.t() @ h.abs() + (dz.abs().t() @ h.abs()) * (half + 2 * len(labels) * U) + half * gw.abs() + tiny
    share = torch.where(g[:, None] == 0, torch.zeros_like(dz), dz / (g * rest)[:, None]).abs().sum(0)
    egw += share[:, None] * 2 * tiny * (g.abs() * rest).max()
    return (gh, gw), (egh * 1.01, egw * 1.01)


@pytest.mark.parametrize("chunks", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_improbable_words(dev, shape, chunks, monkeypatch):
    """Logits of standard deviation 3: most words' probabilities are far below the
    type's least numbers, and so are many gradients but for a loss scale."""
    n, h, v = shape
    hidden, weight, labels, _ = inputs(shape, torch.float32, dev)
    hidden, weight = hidden.half(), (weight * 1.5).half()
    up = torch.randn(n, generator=torch.Generator(device=dev).manual_seed(1), device=dev) * 4096 / n
    if chunks:
        in_chunks(monkeypatch)
    want, bound = exact(hidden, weight, labels, up)
    hidden.requires_grad_(True)
    weight.requires_grad_(True)
    got = torch.autograd.grad(linear_logps(hidden, weight, labels), (hidden, weight), up)
    for x, w, b in zip(got, want, bound):
        near(x, w, b)


@pytest.mark.parametrize("shape", [(64, 128, 2000), (33, 65, 1000)])
def test_a_token_that_the_model_is_sure_of(dev, shape):
    """1 - p of the label near and below the unit roundoff of 32 bits, with logits
    of hundreds: D, whose divisor has lost its bits, stays inside the type."""
    hidden, weight, labels, up = inputs(shape, torch.float16, dev)
    labels[labels == -100] = 3
    toward = weight[labels].float()
    by = torch.linspace(10, 600, shape[0], device=dev)[:, None]
    hidden = (0.05 * hidden.float() + toward * by / toward.square().sum(1, keepdim=True)).half()
    want, bound = logps(hidden, weight, labels, grad=up)
    hidden.requires_grad_(True)
    weight.requires_grad_(True)
    lp = linear_logps(hidden, weight, labels)
    for x, w, b in zip((lp.detach(), *torch.autograd.grad(lp, (hidden, weight), up)), want, bound):
        near(x, w, b)
