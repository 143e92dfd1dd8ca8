"""Token log-probabilities of fp16 operands where the type's range ends."""

import pytest
import torch

from alignment_reference import logps, near
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
