"""Distillation steps, a teacher's log-probabilities and sampled tokens through
SlideFSDP where the output layer has a bias, which goes by torch operations."""

import numpy as np
import pytest
import torch

from alignment_reference import near
from distill_reference import distill
from fullsize import gpu_bf16_copy
from test1_amd.distillation import _torch_distill, linear_top_logps
from test1_amd.sampling import sample_tokens, top_logps
from test_gpu_alignment_e2e import batch, slide
from test_gpu_e2e import V, make_model, u16, units_of

pytestmark = pytest.mark.gpu


def biased():
    model = make_model()
    old, g = model.lm_head, torch.Generator().manual_seed(5)
    model.lm_head = torch.nn.Linear(old.in_features, V, bias=True)
    with torch.no_grad():
        model.lm_head.weight.copy_(old.weight)
        model.lm_head.bias.copy_(torch.randn(V, generator=g))
    return model


def on_gpu(model, dev):
    gm = gpu_bf16_copy(model, dev)
    gm.lm_head.bias = torch.nn.Parameter(model.lm_head.bias.detach().to(dev, torch.bfloat16))
    return gm


@pytest.mark.parametrize("kind,rest", [("forward", True), ("reverse", True), ("forward", False)])
def test_steps(dev, kind, rest):
    model = biased()
    ids, labels, _ = batch(dev)
    g = torch.Generator(device=dev).manual_seed(3)
    teacher = top_logps(torch.randn(4, 95, V, generator=g, device=dev) * 2, 12)
    gm = on_gpu(model, dev).train()
    hidden = gm.model(input_ids=ids, use_cache=False).last_hidden_state[:, :-1]
    mask = labels[:, 1:] != -100
    each = _torch_distill(hidden, gm.lm_head.weight, teacher.ids, teacher.logps, mask, 1 / 1.5, kind, rest, gm.lm_head.bias)
    loss = each.sum() / mask.sum()
    loss.backward()
    # a bias is one more column, of a hidden state that is 1
    wide = torch.cat([hidden.detach(), torch.ones_like(hidden[..., :1])], dim=-1).flatten(0, 1)
    weight = torch.cat([gm.lm_head.weight, gm.lm_head.bias.unsqueeze(1)], dim=1).detach()
    want, bound = distill(wide, weight, teacher.ids.flatten(0, 1), teacher.logps.flatten(0, 1), mask.flatten(), 1 / 1.5, kind, rest)
    sf = slide(dev, model)
    sf.runtime.capture = {}
    out = sf(input_ids=ids, labels=labels, teacher=teacher, temperature=1.5, teacher_kind=kind, teacher_rest=rest)
    sf.wait_for_updates()
    cap, sf.runtime.capture = sf.runtime.capture, None
    near(out.divergences.flatten(), want[0], bound[0])
    assert torch.equal(out.divergences, each.detach()) and torch.equal(out.loss.detach(), loss.detach())
    units = units_of(gm)
    units[-1].append(gm.lm_head.bias)
    for u, ps in enumerate(units):
        assert np.array_equal(u16(cap[u][0]), np.concatenate([u16(p.grad).reshape(-1) for p in ps])), f"unit {u}: gradient"
    sf.close()


def test_words(dev):
    model = biased()
    ids, _, _ = batch(dev)
    gm = on_gpu(model, dev)
    with torch.no_grad():
        hidden = gm.model(input_ids=ids).last_hidden_state
        want = linear_top_logps(hidden[:, :-1], gm.lm_head.weight, 20, 0.8, gm.lm_head.bias)
        logits = torch.mm(hidden[:, -1], gm.lm_head.weight.t(), out_dtype=torch.float32) + gm.lm_head.bias
    sf = slide(dev, model)
    got = sf.top_logps(ids, k=20, temperature=0.8)
    assert torch.equal(got.logps, want.logps) and torch.equal(got.ids, want.ids)
    u = torch.rand(4, generator=torch.Generator().manual_seed(1))
    one, ref = sf.sample_tokens(ids, u, temperature=0.7, top_k=30), sample_tokens(logits, u.to(dev), temperature=0.7, top_k=30)
    assert torch.equal(one.ids, ref.ids) and torch.equal(one.logps, ref.logps)
    sf.close()
