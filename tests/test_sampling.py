"""Token sampling and largest log-probabilities on the CPU: what they compute and
what they refuse."""

import math

import numpy as np
import pytest
import torch

import sampling_reference as reference
from test1_amd import _native
from test1_amd.sampling import TOP_MOST, sample_tokens, top_logps


def rows(kind, n, vocab, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, vocab, generator=g) * 3
    if kind == "ties":
        x = x.round()
    if kind == "masked":
        x[:, vocab // 3:] = -math.inf
    return x


@pytest.mark.parametrize("settings", [{}, dict(temperature=0.7, top_k=5), dict(top_p=0.8), dict(min_p=0.1),
                                      dict(temperature=2.0, top_k=20, top_p=0.6, min_p=0.02), dict(temperature=0.0)])
@pytest.mark.parametrize("kind", ["plain", "ties", "masked"])
def test_draws(kind, settings):
    x = rows(kind, 40, 61)
    u = torch.rand(40, generator=torch.Generator().manual_seed(1))
    out = sample_tokens(x, u, **settings)
    names = dict(t=settings.get("temperature", 1.0), k=settings.get("top_k", 0), p=settings.get("top_p", 1.0),
                 m=settings.get("min_p", 0.0))
    want = [reference.draw(x[i].double().numpy(), float(u[i]), **names) for i in range(40)]
    assert out.ids.tolist() == [w[0] for w in want]
    assert torch.allclose(out.logps.double(), torch.tensor([w[1] for w in want], dtype=torch.float64), rtol=2e-7, atol=1e-7)


def test_settings_of_every_row():
    x = rows("plain", 30, 50)
    g = torch.Generator().manual_seed(2)
    u, t, p, m = torch.rand(30, generator=g), torch.rand(30, generator=g) * 2, torch.rand(30, generator=g) * 1.2, torch.rand(30, generator=g) * 0.1
    k = torch.randint(-1, 30, (30,), generator=g)
    t[3] = 0
    out = sample_tokens(x.view(5, 6, 50), u.view(5, 6), t.view(5, 6), k.view(5, 6), p.view(5, 6), m.view(5, 6))
    assert out.ids.shape == out.logps.shape == (5, 6)
    for i in range(30):
        got = sample_tokens(x[i], u[i], float(t[i]), max(0, int(k[i])), min(1.0, float(p[i])), float(m[i]))
        assert out.ids.view(-1)[i] == got.ids and out.logps.view(-1)[i] == got.logps


@pytest.mark.parametrize("kind", ["plain", "ties", "masked"])
def test_largest(kind):
    x = rows(kind, 9, 300)
    out = top_logps(x.view(3, 3, 300), 128, temperature=1.5)
    assert out.logps.shape == out.ids.shape == (3, 3, 128)
    for i in range(9):
        want = reference.top(x[i].double().numpy(), 128, 1.5)
        assert np.array_equal(out.ids.view(9, 128)[i].numpy(), want[1])
        assert np.allclose(out.logps.view(9, 128)[i].numpy(), want[0], rtol=2e-7, atol=1e-7)


def test_rows_that_are_no_distribution():
    x = rows("plain", 4, 30)
    x[0, 3], x[1, 29], x[2] = math.nan, math.inf, -math.inf
    out, top = sample_tokens(x, torch.full((4,), 0.5)), top_logps(x, 7)
    assert out.ids[:3].tolist() == [-1] * 3 and out.logps[:3].isnan().all() and out.ids[3] >= 0
    assert (top.ids[:3] == -1).all() and top.logps[:3].isnan().all() and top.logps[3].isfinite().all()


def test_uniforms_at_the_ends():
    x = torch.zeros(6, 10)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -1.0, math.nan])
    assert sample_tokens(x, u).ids.tolist() == [0, 9, 9, 9, 0, 0]
    assert sample_tokens(x, u, top_p=0.5).ids.tolist() == [0, 4, 4, 4, 0, 0]   # equal words: the first five
    assert sample_tokens(x, u, top_p=0.0).ids.tolist() == [0] * 6


def test_a_temperature_below_all_that_tells_words_apart():
    x = torch.tensor([[1.0, 3.0, 3.0, 2.0]])
    got = top_logps(x, 4, temperature=1e-45)
    assert got.ids.tolist() == [[1, 2, 3, 0]] and got.logps[0, :2].allclose(torch.tensor(0.5).log())
    assert got.logps[0, 2:].tolist() == [torch.tensor(-1e30).item(), torch.tensor(-2e30).item()]


def test_no_rows_and_no_gradient():
    out = sample_tokens(torch.zeros(0, 5, requires_grad=True), torch.zeros(0))
    assert out.ids.shape == (0,) and not out.logps.requires_grad
    assert top_logps(torch.zeros(2, 0, 5), 3).ids.shape == (2, 0, 3)
    assert not top_logps(torch.zeros(2, 5, requires_grad=True), 3).logps.requires_grad


def test_refusals():
    x, u = torch.zeros(4, 10), torch.zeros(4)
    for bad in (dict(temperature=-1.0), dict(temperature=math.inf), dict(temperature=math.nan), dict(top_k=-1), dict(top_k=1.5),
                dict(top_p=1.1), dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=math.nan), dict(top_p=torch.zeros(3)),
                dict(temperature=torch.zeros(4, 1))):
        with pytest.raises(ValueError):
            sample_tokens(x, u, **bad)
    for bad in (dict(top_k=torch.zeros(4)), dict(top_p=torch.zeros(4, dtype=torch.float64))):
        with pytest.raises(TypeError):
            sample_tokens(x, u, **bad)
    with pytest.raises(ValueError):
        sample_tokens(x, u[:3])
    with pytest.raises(TypeError):
        sample_tokens(x, u.double())
    for f in (lambda t: sample_tokens(t, u), lambda t: top_logps(t, 1)):
        with pytest.raises(TypeError):
            f(x.double())
        with pytest.raises(ValueError):
            f(torch.zeros(4, 0))
    for k in (0, 11, -1):
        with pytest.raises(ValueError):
            top_logps(x, k)
    with pytest.raises(ValueError):
        top_logps(torch.zeros(1, 500), TOP_MOST + 1)
    for t in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            top_logps(x, 2, temperature=t)


def test_entry_points_refuse_without_a_gpu():
    hip = _native.hip()
    assert hip.sf_rows_work(0, 5, 0) == hip.sf_rows_work(5, 0, 0) == hip.sf_rows_work(1, (1 << 30) + 1, 0) == 0
    assert 0 < hip.sf_rows_work(1 << 30, 128_256, _native.SF_DTYPE_BF16) <= 256 << 20
    p = 1 << 20   # never read
    top = lambda logits=p, dtype=0, ld=10, rows=2, vocab=10, k=3, t=1.0, work=p, logps=p, ids=p: hip.sf_top_logps(
        logits, dtype, ld, rows, vocab, k, t, work, logps, ids, None)
    assert top(rows=0) == 0
    for bad in (dict(logits=None), dict(work=None), dict(logps=None), dict(ids=None), dict(ld=9), dict(vocab=0), dict(k=0),
                dict(k=11), dict(k=129, vocab=200, ld=200), dict(t=0.0), dict(t=math.nan), dict(rows=1 << 31)):
        assert top(**bad) == _native.SF_EINVAL, bad
    assert top(dtype=7) == 9003 or top(dtype=7) != 0
    assert top(logits=p + 2) == top(work=p + 8) == _native.SF_EALIGN
    draw = lambda logits=p, rows=2, vocab=10, u=p, work=p, ids=p: hip.sf_sample_tokens(
        logits, 0, 10, rows, vocab, u, 1.0, None, 0, None, 1.0, None, 0.0, None, work, ids, p, None)
    assert draw(rows=0) == 0
    for bad in (dict(logits=None), dict(u=None), dict(work=None), dict(ids=None), dict(vocab=0), dict(vocab=11)):
        assert draw(**bad) == _native.SF_EINVAL, bad
