"""Distillation on the CPU: what it computes and what it refuses."""

import math

import pytest
import torch

from alignment_reference import near
from distill_reference import distill
from test1_amd import _native
from test1_amd.distillation import linear_distill
from test1_amd.sampling import top_logps


def inputs(n, h, v, k, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    hidden = torch.randn(n, h, generator=g).to(dtype)
    weight = (torch.randn(v, h, generator=g) * (2.0 / math.sqrt(h))).to(dtype)
    teacher = top_logps(torch.randn(n, v, generator=g) * 2, k)
    logps = teacher.logps.clone()
    if n > 3 and k > 1:
        logps[1, k // 2:] = -math.inf
        logps[2] = -math.inf
    return hidden, weight, teacher.ids, logps


@pytest.mark.parametrize("kind,rest", [("forward", True), ("forward", False), ("reverse", True)])
@pytest.mark.parametrize("shape", [(1, 8, 5, 1), (9, 16, 40, 7), (9, 16, 12, 12), (5, 24, 300, 128)])
def test_matches_float64(shape, kind, rest):
    hidden, weight, ids, logps = inputs(*shape)
    n = shape[0]
    mask = torch.arange(n) % 4 != 3
    up = torch.randn(n, generator=torch.Generator().manual_seed(1))
    want, bound = distill(hidden, weight, ids, logps, mask, 0.5, kind, rest, grad=up)
    hidden.requires_grad_(True), weight.requires_grad_(True)
    loss = linear_distill(hidden, weight, ids, logps, mask, temperature=2.0, kind=kind, rest=rest)
    for got, w, b in zip((loss.detach(), *torch.autograd.grad(loss, (hidden, weight), up)), want, bound):
        near(got, w, b)


@pytest.mark.parametrize("kind,rest", [("forward", True), ("forward", False), ("reverse", True)])
def test_gradient_against_differences(kind, rest):
    """Central differences of the float64 reference in random directions."""
    hidden, weight, ids, logps = inputs(4, 12, 30, 5)
    up = torch.randn(4, generator=torch.Generator().manual_seed(1))
    _, gh, gw = distill(hidden, weight, ids, logps, None, 1.0, kind, rest, grad=up)[0]
    g = torch.Generator().manual_seed(3)
    for _ in range(3):
        dh, dw = torch.randn(4, 12, generator=g, dtype=torch.float64), torch.randn(30, 12, generator=g, dtype=torch.float64)
        step = 1e-5
        at = lambda s: (distill(hidden.double() + s * dh, weight.double() + s * dw, ids, logps, None, 1.0, kind, rest)[0][0]  # noqa: E731
                        * up.double()).sum()
        slope = (at(step) - at(-step)) / (2 * step)
        assert abs(slope - ((gh * dh).sum() + (gw * dw).sum())) < 1e-7 * (1 + abs(slope))


def test_a_teacher_that_is_the_student():
    """No loss and no gradient where the distributions are the same."""
    hidden, weight, _, _ = inputs(6, 16, 40, 3)
    own = top_logps(hidden @ weight.t(), 10)
    for kind in ("forward", "reverse"):
        hr = hidden.clone().requires_grad_(True)
        loss = linear_distill(hr, weight, own.ids, own.logps, kind=kind)
        assert loss.abs().max() < 1e-6
        # p - q is a rounding of the teacher's log-probabilities, 2^-24 of up to 16, and of the logits
        assert torch.autograd.grad(loss.sum(), hr)[0].abs().max() < 1e-5


def test_words_that_are_wrong():
    hidden, weight, ids, logps = inputs(7, 16, 40, 6)
    ids[0, 0], ids[3, 1], ids[4, 2] = 40, -1, ids[4, 1]
    ids[1, 5] = 1 << 40   # of no word: its log-probability is -infinity
    mask = torch.ones(7, dtype=torch.bool)
    hidden.requires_grad_(True)
    for kind, rest in (("forward", True), ("forward", False), ("reverse", True)):
        loss = linear_distill(hidden, weight, ids, logps, mask, kind=kind, rest=rest)
        assert loss[[0, 3, 4]].isnan().all() and loss[[1, 5, 6]].isfinite().all() and loss[2] == 0
        grad = torch.autograd.grad(loss.sum(), hidden)[0]
        assert grad[[0, 3, 4]].isnan().any(dim=1).all() and grad[[1, 2, 5, 6]].isfinite().all()
    mask[[0, 3, 4]] = False
    assert linear_distill(hidden, weight, ids, logps, mask).isfinite().all()


def test_refusals():
    hidden, weight, ids, logps = inputs(6, 16, 40, 3)
    good = dict(hidden=hidden, weight=weight, teacher_ids=ids, teacher_logps=logps)
    for bad in (dict(weight=weight[:, :8]), dict(teacher_ids=ids[:, :2]), dict(teacher_ids=ids[:5], teacher_logps=logps[:5]),
                dict(teacher_ids=ids[:, :0], teacher_logps=logps[:, :0]), dict(mask=torch.ones(5, dtype=torch.bool)),
                dict(teacher_ids=ids.repeat(1, 43), teacher_logps=logps.repeat(1, 43)), dict(weight=weight[:0]),
                dict(temperature=0.0), dict(temperature=math.inf), dict(kind="both"), dict(kind="reverse", rest=False),
                dict(teacher_logps=logps.clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            linear_distill(**{**good, **bad})
    for bad in (dict(hidden=hidden.double(), weight=weight.double()), dict(weight=weight.bfloat16()), dict(teacher_ids=ids.int()),
                dict(teacher_logps=logps.half()), dict(mask=torch.ones(6))):
        with pytest.raises(TypeError):
            linear_distill(**{**good, **bad})


def test_temperatures_that_leave_fp32():
    hidden, weight, ids, logps = inputs(6, 16, 40, 3)
    for t in (1e-39, 1e39, -1.0, math.nan):
        with pytest.raises(ValueError):
            linear_distill(hidden, weight, ids, logps, temperature=t)
    assert linear_distill(hidden, weight, ids, logps, temperature=1e30).isfinite().all()


def test_shapes_and_no_rows():
    hidden, weight, ids, logps = inputs(12, 16, 40, 3)
    flat = linear_distill(hidden, weight, ids, logps)
    assert torch.equal(linear_distill(hidden.view(3, 4, 16), weight, ids.view(3, 4, 3), logps.view(3, 4, 3)), flat.view(3, 4))
    assert torch.equal(linear_distill(hidden[5], weight, ids[5], logps[5]), flat[5])
    hr, wr = hidden[:0].clone().requires_grad_(True), weight.clone().requires_grad_(True)
    loss = linear_distill(hr, wr, ids[:0], logps[:0])
    gh, gw = torch.autograd.grad(loss.sum(), (hr, wr))
    assert loss.shape == (0,) and gh.shape == (0, 16) and (gw == 0).all()


def test_entry_points_refuse_without_a_gpu():
    hip, p = _native.hip(), 1 << 20   # never read
    E, A = _native.SF_EINVAL, _native.SF_EALIGN
    lists = lambda ids=p, ld=4, rows=2, k=4, vocab=10, words=p: hip.sf_distill_lists(  # noqa: E731
        ids, ld, p, 4, None, rows, k, vocab, 0, words, p, p, p, None)
    assert lists(rows=0) == 0
    assert [lists(**b) for b in (dict(ids=None), dict(ld=3), dict(k=0), dict(k=129), dict(vocab=0), dict(words=None))] == [E] * 6
    tiles = lambda weight=p, ldw=64, h=64, k=4, scale=1.0, dtype=1, keep=None, ldk=0, rows=2, close=0: hip.sf_distill_tiles(  # noqa: E731
        weight, ldw, 300, p, 64, rows, h, p, p, p, k, scale, dtype, p, p, None, keep, ldk, close, None)
    assert tiles(rows=0) == 0
    assert [tiles(**b) for b in (dict(weight=None), dict(ldw=32), dict(h=0), dict(k=0), dict(scale=0.0), dict(scale=math.nan),
                                 dict(keep=p, ldk=300), dict(close=1))] == [E] * 8
    assert [tiles(**b) for b in (dict(weight=p + 2), dict(h=32), dict(ldw=65), dict(keep=p + 8, ldk=512))] == [A] * 4
    assert tiles(dtype=0) not in (0, E)
    loss = lambda parts=p, row=2, form=0, rest=1, scale=1.0, ldh=64, weight=p, dtype=1, slopes=p, stats=p: hip.sf_distill_loss(  # noqa: E731
        parts, row, 0, p, p, p, p, 2, 4, 300, scale, form, rest, p, ldh, weight, 64, 64, dtype, p, p, slopes, stats, 2, None)
    assert [loss(**b) for b in (dict(parts=None), dict(row=1), dict(form=2), dict(form=1, rest=0), dict(scale=-1.0),
                                dict(stats=None), dict(ldh=63), dict(weight=None))] == [E] * 8
    assert loss(weight=p + 2) == loss(ldh=65) == loss(dtype=0) == A and loss(dtype=7) not in (0, E, A)
    by = lambda grad=p, dtype=1, rows=2: hip.sf_distill_weight(grad, p, p, rows, 1.0, dtype, p, p, None)  # noqa: E731
    assert by(rows=0) == 0 and by(grad=None) == E and by(dtype=0) not in (0, E)
    grad = lambda keep=p, ld=512, padded=64, grad=p, dtype=1, norm=p, cleared=0: hip.sf_distill_keep_grad(  # noqa: E731
        keep, ld, 2, padded, 300, p, p, p, p, 4, p, p, 2, dtype, grad, 1.0, norm, None, cleared, None)
    assert grad(padded=0) == 0
    assert [grad(**b) for b in (dict(keep=None), dict(ld=256), dict(padded=1), dict(grad=None), dict(dtype=2, norm=None), dict(cleared=65))] == [E] * 6
    assert grad(keep=p + 8) == grad(ld=520) == A
    rows = lambda logits=p, ld=300, k=4: hip.sf_distill_rows(logits, ld, 2, 300, p, p, k, 1.0, p, p, None)  # noqa: E731
    assert [rows(logits=None), rows(ld=299), rows(k=0)] == [E] * 3 and rows(logits=p + 2) == A
    whole = lambda logits=p, ld=300, grad=p: hip.sf_distill_grad(logits, ld, 2, 300, p, p, p, 4, 1.0, p, p, 2, grad, None)  # noqa: E731
    assert [whole(logits=None), whole(ld=299), whole(grad=None)] == [E] * 3
    turn = lambda hidden=p, ldh=64, ldt=64, order=p: hip.sf_distill_hidden(hidden, ldh, 2, 64, order, p, p, ldt, None)  # noqa: E731
    assert [turn(hidden=None), turn(ldh=63), turn(ldt=128), turn(ldt=63), turn(order=None)] == [E] * 5
    assert turn(hidden=p + 2) == turn(ldh=65) == A
    add = lambda parts=p, done=300, order=p, norm=p, ldw=64, ld=512, live=0: hip.sf_distill_sum(  # noqa: E731
        parts, 1, live, 2, 64, order, p, p, p, norm, p, ld, p, ldw, done, 300, 1, p, None)
    assert [add(parts=None), add(done=301), add(order=None), add(norm=None), add(ldw=63), add(ld=299),
            add(done=299, live=1)] == [E] * 7
    assert add(ldw=65) == add(parts=p + 8) == A
    assert hip.sf_distill_hidden_product(p, 512, 2, None, p, 64, 300, 64, 1, p, 1, None) == E
    assert hip.sf_distill_weight_grad(p, 512, 64, None, 300, p, 64, None, 1, p, None) == E
