"""Token sampling and largest log-probabilities on the GPU where logits over the
temperature are large: masks of finite values over whole parts of a row, low
temperatures; and all kinds of rows over several parts."""

import numpy as np
import pytest
import torch

import sampling_reference as reference
from test1_amd.sampling import sample_tokens, top_logps
from test_gpu_sampling import KINDS, SETTINGS, against, close, rows

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
# of up to 16,384 words of 16 bits or 8,192 of 32 a row is one part; these have 1, 3 and 5, and 8 and 16
LENGTHS = [700, 40_003, 128_256]


def largest_are(x, k, t):
    out = top_logps(x, k, temperature=t)
    for i in range(x.shape[0]):
        logps, ids = reference.top(x[i].double().cpu().numpy(), k, t)
        assert np.array_equal(out.ids[i].cpu().numpy(), ids), (k, t)
        assert all(close(a, b) for a, b in zip(out.logps[i].double().cpu().numpy(), logps)), (k, t)


def draws_are(x, g, **s):
    u = torch.rand(x.shape[0], generator=g, device=x.device)
    out = sample_tokens(x, u, s.get("t", 1.0), s.get("k", 0), s.get("p", 1.0), s.get("m", 0.0))
    against(x, u.cpu(), out, **s)
    # the same by settings of every row
    every = lambda name, least, kind: torch.full_like(u, s.get(name, least), dtype=kind)  # noqa: E731
    own = sample_tokens(x, u, every("t", 1.0, torch.float32), every("k", 0, torch.int64), every("p", 1.0, torch.float32),
                        every("m", 0.0, torch.float32))
    settings = {n: (v if n == "k" else float(torch.tensor(v))) for n, v in s.items()}
    against(x, u.cpu(), own, **settings)


@pytest.mark.parametrize("t", [1.0, 0.3, 0.1])
@pytest.mark.parametrize("mask", [-3e4, -1e9, -1e10, -1e12, -1e20, -1e30])
@pytest.mark.parametrize("vocab", LENGTHS)
def test_whole_parts_of_a_finite_mask(dev, vocab, mask, t):
    """A few hundred neighbouring words are allowed, fewer than asked for in one row, none in the last: the
    others hold a mask's value, whole parts of it."""
    g = torch.Generator(device=dev).manual_seed(vocab)
    for dtype in TYPES:
        if abs(mask) > torch.finfo(dtype).max:
            continue
        x = torch.full((3, vocab), mask, device=dev)
        x[0, vocab // 2:vocab // 2 + 300] = torch.randn(300, generator=g, device=dev) * 2.5
        x[1, vocab // 3:vocab // 3 + 5] = torch.randn(5, generator=g, device=dev)
        x = x.to(dtype)
        for k in (1, 20, 128):
            largest_are(x, k, t)
        for s in (dict(t=0.0), dict(t=t, k=1), dict(t=t, k=50, p=0.95), dict(t=t, k=128), dict(t=t, k=128, m=0.01),
                  dict(t=t, k=300), dict(t=t, p=0.9), dict(t=t, m=0.05), dict(t=t)):
            draws_are(x, g, **s)


@pytest.mark.parametrize("t", [0.3, 0.02, 1e-3, 1e-6, 1e-8, 1e-9, 1e-10, 1e-12, 1e-20, 1e-30])
@pytest.mark.parametrize("vocab", LENGTHS)
def test_low_temperatures(dev, vocab, t):
    t = max(float(torch.tensor(t)), 1e-30)   # what fp32 settings hold of it
    g = torch.Generator(device=dev).manual_seed(vocab)
    for dtype in TYPES:
        x = rows("plain", 3, vocab, dtype, dev, seed=1)
        x[1] += 300.0
        x[2] -= 3000.0
        for k in (1, 20, 128):
            largest_are(x, k, t)
        for s in (dict(t=t, k=1), dict(t=t, k=50, p=0.95), dict(t=t, k=128, m=0.01), dict(t=t, k=300), dict(t=t, p=0.9), dict(t=t)):
            draws_are(x, g, **s)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40_003, 128_256, 270_001])
def test_all_kinds_of_rows_over_several_parts(dev, vocab, dtype):
    g = torch.Generator(device=dev).manual_seed(vocab)
    for kind in KINDS:
        x = rows(kind, 2, vocab, dtype, dev, seed=7)
        for s in SETTINGS if vocab < 200_000 else SETTINGS[2:10:2]:
            u = torch.rand(2, generator=g, device=dev)
            out = sample_tokens(x, u, s.get("t", 1.0), s.get("k", 0), s.get("p", 1.0), s.get("m", 0.0))
            against(x, u.cpu(), out, **s)


@pytest.mark.parametrize("t", [20.0, 1e4, 1e30])
@pytest.mark.parametrize("vocab", LENGTHS)
def test_high_temperatures(dev, vocab, t):
    t = float(torch.tensor(t))
    g = torch.Generator(device=dev).manual_seed(vocab)
    for dtype in TYPES:
        x = rows("plain", 2, vocab, dtype, dev, seed=2)
        x[1, vocab // 4:] = float("-inf")
        for k in (1, 128):
            largest_are(x, k, t)
        for s in (dict(t=t, k=50, p=0.95), dict(t=t, k=300), dict(t=t, p=0.93), dict(t=t, m=0.5), dict(t=t)):
            draws_are(x, g, **s)


def test_other_modes_and_settings(dev):
    """Under inference mode and autocast, of logits with a gradient, settings beyond the vocabulary."""
    x = rows("plain", 5, 40_003, torch.bfloat16, dev)
    u = torch.rand(5, device=dev)
    want, top = sample_tokens(x, u, top_p=0.9), top_logps(x, 30)
    same = lambda a, b: all(torch.equal(p, q) for p, q in zip(a, b))  # noqa: E731
    with torch.inference_mode():
        assert same(sample_tokens(x.clone(), u, top_p=0.9), want) and same(top_logps(x, 30), top)
    with torch.autocast("cuda", dtype=torch.float16):
        assert same(sample_tokens(x, u, top_p=0.9), want)
    out = top_logps(torch.nn.Parameter(x), 30)
    assert same(out, top) and not out.logps.requires_grad
    assert same(sample_tokens(x, u, top_k=1 << 40), sample_tokens(x, u))
    assert same(sample_tokens(x, u, top_k=torch.full((5,), 1 << 40, device=dev)), sample_tokens(x, u, top_k=torch.zeros(5, dtype=torch.int64, device=dev)))
    for s in (dict(temperature=torch.tensor(0.7)), dict(temperature=torch.tensor(0.7, device=dev)), dict(top_k=torch.tensor(40))):
        assert same(sample_tokens(x, u, **s), sample_tokens(x, u, **{n: v.item() for n, v in s.items()}))
