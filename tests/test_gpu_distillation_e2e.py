"""Distillation steps, a teacher's log-probabilities and sampled tokens through
SlideFSDP: losses and gradients bit-identical to non-offloaded runs that compute
the same."""

import math

import numpy as np
import pytest
import torch

from fullsize import gpu_bf16_copy
from test1_amd.distillation import linear_distill, linear_top_logps
from test1_amd.sampling import TopLogps, sample_tokens, top_logps
from test_gpu_alignment_e2e import batch, slide
from test_gpu_e2e import L, V, make_model, u16, units_of

pytestmark = pytest.mark.gpu


def non_offloaded(model, dev, ids, labels, loss_of):
    """(loss, divergences, gradients of the units)"""
    gm = gpu_bf16_copy(model, dev)
    gm.train()
    hidden = gm.model(input_ids=ids, use_cache=False).last_hidden_state
    each = loss_of(hidden[:, :-1], gm.lm_head.weight, labels[:, 1:] != -100)
    loss = each.sum() / (labels[:, 1:] != -100).sum()
    loss.backward()
    return loss.detach(), each.detach(), [np.concatenate([u16(p.grad).reshape(-1) for p in ps]) for ps in units_of(gm)]


@pytest.mark.parametrize("kind,rest,resident", [("forward", True, 0), ("reverse", True, L - 1), ("forward", False, L - 1)])
def test_step_equals_the_non_offloaded_one(dev, kind, rest, resident):
    model = make_model()
    ids, labels, _ = batch(dev)
    g = torch.Generator(device=dev).manual_seed(3)
    teacher = top_logps(torch.randn(4, 95, V, generator=g, device=dev) * 2, 12)
    want = non_offloaded(model, dev, ids, labels,
                         lambda h, w, m: linear_distill(h, w, teacher.ids, teacher.logps, m, 1.5, kind, rest))
    sf = slide(dev, model, resident_layers=resident)
    sf.runtime.capture = {}
    out = sf(input_ids=ids, labels=labels, teacher=TopLogps(teacher.logps.cpu(), teacher.ids.cpu()), temperature=1.5,
             teacher_kind=kind, teacher_rest=rest)
    sf.wait_for_updates()
    cap, sf.runtime.capture = sf.runtime.capture, None
    assert torch.equal(out.loss.detach(), want[0]) and torch.equal(out.divergences, want[1])
    for u, ref in enumerate(want[2]):
        assert np.array_equal(u16(cap[u][0]), ref), f"unit {u}: gradient"
    # an objective of the divergences; without labels every token counts
    seen = {}

    def objective(each, mask):
        seen.update(each=each.detach(), mask=mask)
        return (each * mask).square().mean(), each.sum()

    out = sf(input_ids=ids, teacher=teacher, objective=objective)
    assert out.loss.isfinite() and bool(seen["mask"].all()) and torch.equal(out.divergences, seen["each"])
    assert sf(input_ids=ids, labels=labels).loss.isfinite()
    sf.close()


def test_teacher_and_sampled_tokens(dev):
    model = make_model()
    ids, labels, _ = batch(dev)
    gm = gpu_bf16_copy(model, dev)
    with torch.no_grad():
        hidden = gm.model(input_ids=ids).last_hidden_state
        want = linear_top_logps(hidden[:, :-1], gm.lm_head.weight, 20, 0.8)
    sf = slide(dev, model)
    got = sf.top_logps(ids, k=20, temperature=0.8)
    assert torch.equal(got.logps, want.logps) and torch.equal(got.ids, want.ids)
    # a student that is its own teacher
    assert sf(input_ids=ids, labels=labels, teacher=sf.top_logps(ids, k=20)).loss.abs() < 1e-4
    fresh = make_model()
    sf.close()
    sf = slide(dev, fresh)
    u = torch.rand(4, generator=torch.Generator().manual_seed(1))
    one = sf.sample_tokens(ids, u, temperature=0.7, top_p=0.9)
    with torch.no_grad():
        logits = torch.mm(hidden[:, -1], gm.lm_head.weight.t(), out_dtype=torch.float32)
    ref = sample_tokens(logits, u.to(dev), temperature=0.7, top_p=0.9)
    assert torch.equal(one.ids, ref.ids) and torch.equal(one.logps, ref.logps)
    # its log-probability is that of the label there, of the same forward: the last column is masked
    mask = torch.ones_like(ids)
    mask[:, -1] = 0
    one_back = sf.sample_tokens(ids, u, attention_mask=mask, temperature=0.7, top_k=40)
    drawn = ids.clone()
    drawn[:, -1] = one_back.ids
    lp = sf.token_logps(ids, attention_mask=mask, labels=drawn, temperature=0.7)[:, -1]
    # two products of 256 terms in fp32 and two sums of exponentials, each within 1024 U of magnitudes up to 20
    assert (lp - one_back.logps).abs().max() <= 2 * 1024 * 2.0 ** -24 * 20
    # padded rows: behind the last token that is there
    mask = torch.ones_like(ids)
    mask[1, 40:] = 0
    short = sf.sample_tokens(ids, u.to(dev), attention_mask=mask, temperature=0.0)
    top = sf.top_logps(ids, attention_mask=mask, k=1)
    assert short.ids[1] == top.ids[1, 39, 0] and (short.logps[1] - top.logps[1, 39, 0]).abs() <= 2 * 1024 * 2.0 ** -24 * 20
    # settings of every row
    own = sf.sample_tokens(ids, u, temperature=torch.tensor([0.7] * 4), top_p=torch.tensor([0.9] * 4))
    assert torch.equal(own.ids, one.ids)
    sf.close()


def test_refusals_before_a_decoder_runs(dev):
    model = make_model()
    ids, labels, _ = batch(dev)
    sf = slide(dev, model)
    good = TopLogps(torch.full((4, 95, 3), -2.0, device=dev), torch.arange(3, device=dev).expand(4, 95, 3))
    for bad in (dict(teacher=TopLogps(good.logps[:, :-1], good.ids[:, :-1])), dict(temperature=0.0), dict(teacher_kind="both"),
                dict(teacher_kind="reverse", teacher_rest=False), dict(labels=labels[:, :-1]),
                dict(teacher=TopLogps(good.logps.expand(4, 95, 3).repeat(1, 1, 43), good.ids.repeat(1, 1, 43)))):
        with pytest.raises(ValueError):
            sf(**{**dict(input_ids=ids, labels=labels, teacher=good), **bad})
    for bad in (good.ids, (good.logps,), TopLogps(good.ids, good.ids)):
        with pytest.raises(TypeError):
            sf(input_ids=ids, teacher=bad)
    for bad in (dict(k=0), dict(k=129), dict(temperature=math.inf)):
        with pytest.raises(ValueError):
            sf.top_logps(ids, **bad)
    u = torch.rand(4)
    for bad in (dict(uniforms=u[:3]), dict(top_p=2.0), dict(attention_mask=torch.ones(4, 5))):
        with pytest.raises(ValueError):
            sf.sample_tokens(**{**dict(input_ids=ids, uniforms=u), **bad})
    assert sf(input_ids=ids, labels=labels, teacher=good).loss.isfinite()
    sf.close()


def test_command(dev):
    from test1_amd.distillation_step import main

    losses = main(["--steps", "2", "--rows", "3", "--prompt", "20", "--length", "2", "--words", "8"])
    assert len(losses) == 2 and all(math.isfinite(x) and x >= 0 for x in losses)
