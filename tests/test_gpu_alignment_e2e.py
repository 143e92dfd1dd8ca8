"""Preference and policy steps through SlideFSDP, and its checkpoints in 8
bits: losses and gradients bit-identical to non-offloaded runs that compute
the same (with 8-bit checkpoints, ones whose recompute reads the restored
input)."""


import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from fullsize import gpu_bf16_copy
from test1_amd.act8 import pack_act8, unpack_act8
from test1_amd.alignment import policy_loss, preference_loss
from test1_amd.linear_logps import linear_logps
from test1_amd import kernels, sliding_checkpoint
from test1_amd.pinned import pinned_empty
from test1_amd.sliding_checkpoint import ActivationRing, KeptOnDevice, SlidingCheckpoint, StorageSpill
from test_gpu_e2e import L, LR, V, WD, make_model, u16, units_of

pytestmark = pytest.mark.gpu


def batch(dev, rows=4, length=96):
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, V, (rows, length), generator=g)
    labels = ids.clone()
    labels[:, :20] = -100          # prompts
    labels[0, 70:] = labels[rows - 1, 50:] = -100
    return ids.to(dev), labels.to(dev), (0.1 * torch.randn(rows, length - 1, generator=g)).to(dev)


def objectives(noise, base, labels):
    other = base + noise
    adv = noise[:, 0] * 10
    return {"preference": lambda lp, m: preference_loss(lp, other, m, beta=0.5),
            "policy": lambda lp, m: policy_loss(lp, other, adv, m, base - noise, kl_coef=0.1, reduction="sequence")}


def slide(dev, model, cfg_kw={}, **kw):
    from test1_amd import SlideFSDP, SlideFSDPConfig

    return SlideFSDP(model, SlideFSDPConfig(device=dev, lr=LR, weight_decay=WD, **cfg_kw), wait_timeout=120, **kw)


class RecomputeFrom8Bits(torch.autograd.Function):
    """A layer whose backward runs it again on its restored input."""

    @staticmethod
    def forward(ctx, x, run, fmt, *params):
        ctx.save_for_backward(x.detach(), *params)
        ctx.run, ctx.fmt = run, fmt
        return run(x.detach())

    @staticmethod
    def backward(ctx, g):
        x, *params = ctx.saved_tensors
        x = unpack_act8(pack_act8(x, ctx.fmt), x.shape, x.dtype, ctx.fmt).requires_grad_(True)
        with torch.enable_grad():
            y = ctx.run(x)
        gx, *gp = torch.autograd.grad(y, (x, *params), g)
        return (gx, None, None, *gp)


def non_offloaded(model, dev, ids, labels, objective, fmt=None):
    """(loss, log-probabilities, gradients of the units)"""
    gm = gpu_bf16_copy(model, dev)
    gm.train()
    if fmt is not None:
        for layer in gm.model.layers[:-1]:
            run = layer.forward

            def forward(h, _run=run, _layer=layer, **kw):
                first = lambda x: (lambda o: o[0] if isinstance(o, tuple) else o)(_run(x, **kw))  # noqa: E731
                return RecomputeFrom8Bits.apply(h, first, fmt, *_layer.parameters())

            layer.forward = forward
    hidden = gm.model(input_ids=ids, use_cache=False).last_hidden_state
    lp = linear_logps(hidden[:, :-1], gm.lm_head.weight, labels[:, 1:])
    loss = objective(lp, labels[:, 1:] != -100).loss
    loss.backward()
    return loss.detach(), lp.detach(), [np.concatenate([u16(p.grad).reshape(-1) for p in ps]) for ps in units_of(gm)]


def check_step(sf, ids, labels, objective, want):
    loss, lp, grads = want
    sf.runtime.capture = {}
    out = sf(input_ids=ids, labels=labels, objective=objective)
    sf.wait_for_updates()
    cap, sf.runtime.capture = sf.runtime.capture, None
    assert torch.equal(out.loss.detach(), loss) and torch.equal(out.logps, lp) and torch.equal(out.result.loss, loss)
    for u, ref in enumerate(grads):
        assert np.array_equal(u16(cap[u][0]), ref), f"unit {u}: gradient"


@pytest.mark.parametrize("what", ["preference", "policy"])
@pytest.mark.parametrize("resident", [0, L - 1])
def test_objective_step_equals_the_non_offloaded_one(dev, what, resident):
    model = make_model()
    ids, labels, noise = batch(dev)
    gm = gpu_bf16_copy(model, dev)
    with torch.no_grad():
        base = linear_logps(gm.model(input_ids=ids).last_hidden_state[:, :-1], gm.lm_head.weight, labels[:, 1:])
    del gm
    objective = objectives(noise, base, labels)[what]
    want = non_offloaded(model, dev, ids, labels, objective)
    sf = slide(dev, model, resident_layers=resident)
    got = sf.token_logps(ids, labels=labels)
    assert torch.equal(got, base) and not got.requires_grad
    check_step(sf, ids, labels, objective, want)
    # the updated model is another policy, and a plain step still runs
    after = sf.token_logps(ids, labels=labels)
    assert not torch.equal(after, base) and after.isfinite().all()
    assert sf(input_ids=ids, labels=labels).loss.isfinite()
    sf.close()


@pytest.mark.parametrize("fmt,cfg,kw", [("int8", {}, {}), ("fp8", {}, dict(resident_layers=0)),
                                        ("int8", {}, dict(checkpoint_d2h="kernel")),
                                        ("int8", dict(ac_offload_mode="nvme"), {})])
def test_step_with_8_bit_checkpoints(dev, fmt, cfg, kw, tmp_path):
    model = make_model()
    ids, labels, noise = batch(dev)
    objective = objectives(noise, torch.full_like(noise, -7.0), labels)["preference"]
    want = non_offloaded(model, dev, ids, labels, objective, fmt)
    exact = non_offloaded(model, dev, ids, labels, objective)
    assert torch.equal(want[0], exact[0])   # the loss is the forward's
    for a, b in zip(want[2], exact[2]):
        a, b = (torch.from_numpy(x.view(np.int16).copy()).view(torch.bfloat16).float() for x in (a, b))
        assert torch.nn.functional.cosine_similarity(a, b, dim=0) > 0.99
    if cfg:
        cfg = dict(cfg, ac_offload_dir=str(tmp_path))
    sf = slide(dev, model, cfg, checkpoint_format=fmt, **kw)
    check_step(sf, ids, labels, objective, want)
    if not cfg:
        assert all(t[0].dtype == torch.int16 and t[0].numel() == 66 * (4 * 96 * 256 // 128) for t in sf.layer_tensors)
    # another batch shape, then the first again
    for n in (64, 96):
        assert sf(input_ids=ids[:2, :n], labels=labels[:2, :n]).loss.isfinite()
    sf.close()


def test_checkpoint_format_refusals(dev):
    from test1_amd import SlideFSDP, SlideFSDPConfig

    with pytest.raises(ValueError, match="format"):
        slide(dev, make_model(), checkpoint_format="int4")
    with pytest.raises(ValueError, match="offloaded"):
        slide(dev, make_model(), dict(ac_offload_mode="none"), checkpoint_format="int8")
    with pytest.raises(ValueError, match="pin_memory"):
        SlidingCheckpoint(layer_idx=1, layer_tensors=[[]], pin_memory=False, checkpoint_format="int8")
    sf = slide(dev, make_model())
    with pytest.raises(ValueError, match="labels"):
        sf(input_ids=torch.zeros(2, 8, dtype=torch.int64, device=dev), objective=lambda lp, m: lp.sum())
    sf.close()


@pytest.mark.parametrize("mode", ["host", "host_sdma", "storage", "kept"])
@pytest.mark.parametrize("use_ring", [True, False])
def test_masks_stay_exact_and_hidden_states_come_back_restored(dev, mode, use_ring, tmp_path, monkeypatch):
    """Every layer but the last recomputes from the restored hidden states; its
    mask, a second checkpoint tensor, is what it was."""
    n, shape = 5, (2, 33, 200)
    if mode == "host_sdma":
        kernels.dma_init(dev)
    if mode == "kept":
        monkeypatch.setattr(sliding_checkpoint, "pin_or_keep", KeptOnDevice)
    spill = StorageSpill(n_slots=3) if mode == "storage" else None
    paths = [[f"{tmp_path}/a-{i}-{c}.bin" for c in range(4)] for i in range(n)]
    slots = [[] for _ in range(n)]
    ring = ActivationRing(dev) if use_ring else None
    mask = (torch.rand(shape, generator=torch.Generator().manual_seed(4)) < 0.3).to(dev)
    seen = {}

    def layer(x, i, m):
        seen.setdefault(i, []).append((x.detach().clone(), m.clone()))
        return torch.tanh(x * 1.1).masked_fill(m, 0.0)

    x = torch.randn(shape, generator=torch.Generator().manual_seed(0)).bfloat16().to(dev).requires_grad_(True)
    for i in range(n):
        with SlidingCheckpoint(layer_idx=i + 1, layer_tensors=slots, gds_offload=mode == "storage", file_paths=paths,
                               is_last_layer=i == n - 1, device=str(dev), prefetch_ring=ring, spill=spill,
                               pack_engine="sdma" if mode == "host_sdma" else "kernel", checkpoint_format="int8"):
            h = x if i == 0 else h
            h = checkpoint(layer, h, i, mask, use_reentrant=False)
    h.float().sum().backward()
    torch.cuda.synchronize()
    for i in range(n):
        (a, ma), (b, mb) = seen[i]
        want = a if i == n - 1 else unpack_act8(pack_act8(a), a.shape, a.dtype)
        assert torch.equal(b, want) and torch.equal(ma, mb), i
    if ring is not None:
        ring.close()
    if spill is not None:
        spill.close()


def test_the_example_learns(dev):
    from test1_amd.preference_step import main

    losses = main(["--steps", "3", "--pairs", "2", "--length", "64"])
    assert len(losses) == 6 and all(np.isfinite(losses))
    assert losses[2] < losses[0] and losses[5] < losses[3]


class _Own(Exception):
    """An objective's own error."""


def _raise(lp, mask):
    raise _Own


def test_errors_behind_the_decoders_give_the_units_back(dev, monkeypatch):
    """Two pool units and no unit with a buffer of its own: whatever raises
    between the decoders and the backward, the next step is that of a trainer
    where nothing had raised."""
    from test1_amd import SlideFSDP, SlideFSDPConfig, slide_fsdp

    model = make_model()
    ids, labels, noise = batch(dev)
    objective = objectives(noise, torch.full_like(noise, -7.0), labels)["preference"]
    want = non_offloaded(model, dev, ids, labels, objective)
    base = want[1]
    sf = SlideFSDP(model, SlideFSDPConfig(device=dev, lr=LR, weight_decay=WD), wait_timeout=10, resident_layers=0)
    for bad, error in ((_raise, _Own), (lambda lp, m: objective(lp[:, 1:], m), ValueError),
                       (lambda lp, m: objective(lp, m).loss.detach(), RuntimeError)):
        with pytest.raises(error):
            sf(input_ids=ids, labels=labels, objective=bad)
        assert torch.equal(sf.token_logps(ids, labels=labels), base)

    def failing(*args):
        raise _Own

    with monkeypatch.context() as m:
        m.setattr(slide_fsdp, "linear_logps", failing)
        for call in (lambda: sf.token_logps(ids, labels=labels),
                     lambda: sf(input_ids=ids, labels=labels, objective=objective)):
            with pytest.raises(_Own):
                call()
    with monkeypatch.context() as m:
        m.setattr(sf.output_layer, "forward", failing)
        with pytest.raises(_Own):
            sf(input_ids=ids, labels=labels)
    check_step(sf, ids, labels, objective, want)
    sf.close()


def test_calls_refused_before_a_decoder_runs(dev, monkeypatch):
    sf = slide(dev, make_model())
    ids, labels, _ = batch(dev)

    def ran(*args):
        raise AssertionError("the decoders ran")

    monkeypatch.setattr(sf, "_run_decoders", ran)
    mean = lambda lp, m: -lp[m].mean()  # noqa: E731
    for kw, error in ((dict(temperature=0.0), ValueError), (dict(temperature=float("nan")), ValueError),
                      (dict(labels=labels[:, 1:]), ValueError), (dict(labels=labels.int()), TypeError)):
        kw = dict(dict(labels=labels), **kw)
        with pytest.raises(error):
            sf.token_logps(ids, **kw)
        with pytest.raises(error):
            sf(input_ids=ids, objective=mean, **kw)
    sf.close()


def test_an_objective_that_returns_a_tuple(dev):
    model = make_model()
    ids, labels, noise = batch(dev)
    objective = objectives(noise, torch.full_like(noise, -7.0), labels)["preference"]
    want = non_offloaded(model, dev, ids, labels, objective)
    sf = slide(dev, model)
    with pytest.raises(TypeError, match="objective returns"):
        sf(input_ids=ids, labels=labels, objective=lambda lp, m: None)
    sf.runtime.capture = {}
    out = sf(input_ids=ids, labels=labels, objective=lambda lp, m: (objective(lp, m).loss, {"tokens": int(m.sum())}))
    sf.wait_for_updates()
    cap, sf.runtime.capture = sf.runtime.capture, None
    assert torch.equal(out.loss.detach(), want[0]) and out.result[1]["tokens"] == int((labels[:, 1:] != -100).sum())
    for u, ref in enumerate(want[2]):
        assert np.array_equal(u16(cap[u][0]), ref), u
    sf.close()
