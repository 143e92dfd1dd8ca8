"""Token log-probabilities, the losses over them and 8-bit checkpoints on the
host: the formulas against float64, gradients against differences, refusals."""

import math

import pytest
import torch

from alignment_reference import logps, near, policy, preference
from test1_amd.act8 import act8_bytes, pack_act8, unpack_act8
from test1_amd.alignment import policy_loss, preference_loss
from test1_amd.linear_logps import linear_logps


def tokens(shape=(4, 37), seed=0):
    g = torch.Generator().manual_seed(seed)
    mask = torch.rand(shape, generator=g) < 0.7
    mask[1] = False
    lp = -3 * torch.rand(shape, generator=g)
    noise = lambda: torch.randn(shape, generator=g)  # noqa: E731
    return mask, lp, lp + 0.2 * noise(), lp + 0.3 * noise(), noise()


@pytest.mark.parametrize("kind,smoothing,average", [("sigmoid", 0.0, False), ("sigmoid", 0.1, True), ("hinge", 0.0, False),
                                                    ("ipo", 0.0, True)])
def test_preference(kind, smoothing, average):
    mask, lp, ref, _, _ = tokens()
    want, bound = preference(lp, ref, mask, 0.1, kind, smoothing, average)
    lp = torch.where(mask, lp, torch.full_like(lp, math.nan)).requires_grad_(True)
    out = preference_loss(lp, ref, mask, 0.1, kind, smoothing, average)
    grad = torch.autograd.grad(out.loss, lp)[0]
    for got, w, b in zip((out.loss.detach(), out.chosen_rewards, out.rejected_rewards, grad), want, bound):
        near(got, w, 16 * b + 1e-6 * w.abs())   # torch adds all of a row in 32 bits


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("with_ref", [False, True])
def test_policy(with_ref, reduction):
    mask, lp, old, ref, adv = tokens()
    ref = ref if with_ref else None
    want, bound = policy(lp, old, adv, mask, ref, 0.2, 0.28, 0.05, reduction)
    old = torch.where(mask, old, torch.full_like(old, -math.inf))
    lp.requires_grad_(True)
    out = policy_loss(lp, old, adv, mask, ref, 0.2, 0.28, 0.05, reduction)
    grad = torch.autograd.grad(out.loss, lp)[0]
    near(out.loss.detach(), want[0], 16 * bound[0])
    near(grad, want[3], 16 * bound[3])
    assert (out.kl is None) != with_ref
    near(out.clip_fraction, want[2], 16 * bound[2])


def test_logps_and_gradients_against_differences():
    g = torch.Generator().manual_seed(3)
    hidden, weight = torch.randn(9, 12, generator=g), torch.randn(31, 12, generator=g)
    labels = torch.randint(0, 31, (9,), generator=g)
    labels[2] = -100
    up = torch.randn(9, generator=g)
    want, bound = logps(hidden, weight, labels, 1 / 0.7, grad=up)
    h, w = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    lp = linear_logps(h, w, labels, temperature=0.7)
    for got, x, b in zip((lp.detach(), *torch.autograd.grad(lp, (h, w), up)), want, bound):
        near(got, x, b)
    step = 2.0 ** -6
    for i, j in ((0, 0), (4, 7), (8, 11)):
        hi, lo = hidden.double().clone(), hidden.double().clone()
        hi[i, j] += step
        lo[i, j] -= step
        diff = ((logps(hi, weight, labels, 1 / 0.7)[0][0] - logps(lo, weight, labels, 1 / 0.7)[0][0]) * up).sum() / (2 * step)
        assert abs(diff - want[1][i, j]) <= 0.01 * (abs(want[1][i, j]) + 0.1)   # third derivatives times step^2
    assert linear_logps(hidden, weight, torch.full((9,), 31))[0].isnan()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("shape", [(1,), (3, 77), (2, 5, 128), (0, 4)])
def test_checkpoint_round_trip(shape, fmt):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).bfloat16()
    packed = pack_act8(x, fmt)
    assert packed.dtype == torch.uint8 and packed.numel() == act8_bytes(x.numel())
    back = unpack_act8(packed, shape, x.dtype, fmt)
    assert back.shape == x.shape and ((back - x).abs() <= 0.08 * x.abs() + 0.02).all()
    out = torch.empty_like(x)
    assert unpack_act8(packed, shape, x.dtype, fmt, out=out) is out and torch.equal(out, back)


def test_refusals():
    mask, lp, old, ref, adv = tokens()
    bad = [
        (ValueError, lambda: preference_loss(lp[:3], ref[:3], mask[:3])),
        (ValueError, lambda: preference_loss(lp, ref[:, :5], mask)),
        (ValueError, lambda: preference_loss(lp, ref, mask[:, :5])),
        (TypeError, lambda: preference_loss(lp, ref, mask.int())),
        (TypeError, lambda: preference_loss(lp.bfloat16(), ref, mask)),
        (ValueError, lambda: preference_loss(lp, ref, mask, beta=0.0)),
        (ValueError, lambda: preference_loss(lp, ref, mask, kind="dpo")),
        (ValueError, lambda: preference_loss(lp, ref, mask, kind="ipo", label_smoothing=0.1)),
        (ValueError, lambda: preference_loss(lp, ref.requires_grad_(True), mask)),
        (ValueError, lambda: preference_loss(lp[0], ref.detach()[0], mask[0])),
        (ValueError, lambda: policy_loss(lp, old, adv[:, :3], mask)),
        (ValueError, lambda: policy_loss(lp, old, adv, mask, clip_low=1.5)),
        (ValueError, lambda: policy_loss(lp, old, adv, mask, clip_high=-0.1)),
        (ValueError, lambda: policy_loss(lp, old, adv, mask, reduction="mean")),
        (TypeError, lambda: policy_loss(lp, old.double(), adv, mask)),
        (ValueError, lambda: policy_loss(lp, old, adv, mask, kl_coef=math.nan)),
        (ValueError, lambda: linear_logps(torch.zeros(2, 3), torch.zeros(5, 4), torch.zeros(2).long())),
        (ValueError, lambda: linear_logps(torch.zeros(2, 4), torch.zeros(5, 4), torch.zeros(3).long())),
        (TypeError, lambda: linear_logps(torch.zeros(2, 4), torch.zeros(5, 4).bfloat16(), torch.zeros(2).long())),
        (TypeError, lambda: linear_logps(torch.zeros(2, 4), torch.zeros(5, 4), torch.zeros(2).int())),
        (ValueError, lambda: linear_logps(torch.zeros(2, 4), torch.zeros(5, 4), torch.zeros(2).long(), temperature=0.0)),
        (ValueError, lambda: linear_logps(torch.zeros(2, 4), torch.zeros(0, 4), torch.zeros(2).long())),
        (ValueError, lambda: pack_act8(lp, "int4")),
        (TypeError, lambda: pack_act8(lp.double())),
        (ValueError, lambda: pack_act8(lp, out=torch.empty(3, dtype=torch.uint8))),
        (ValueError, lambda: unpack_act8(torch.empty(100, dtype=torch.uint8), (77,))),
        (TypeError, lambda: unpack_act8(torch.empty(132, dtype=torch.uint8), (77,), torch.float64)),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {i} was taken")


def test_c_entry_points_refuse_without_a_gpu():
    from test1_amd import _native

    hip = _native.hip()
    one = 64   # an address that is never read: each call ends at its check
    assert hip.sf_logps_rows(None, 8, 1, 8, one, -100, 1.0, one, one, None) == 9001
    assert hip.sf_logps_rows(one, 6, 1, 8, one, -100, 1.0, one, one, None) == 9001
    assert hip.sf_logps_rows(one, 9, 1, 8, one, -100, 1.0, one, one, None) == 9007
    assert hip.sf_logps_rows(one, 8, 0, 8, one, -100, 1.0, one, one, None) == 0
    assert hip.sf_logps_grad(one, 8, 1, 8, one, -100, 1.0, one, one, one, one, 7, 8, None) == 9003
    assert hip.sf_logps_grad(one, 8, 1, 8, one, -100, 1.0, one, one, one, one, 1, 8, None) == 9005
    assert hip.sf_logps_weight(None, one, one, -100, 1, 8, 1.0, one, None, None) == 9001
    tiles = lambda **k: hip.sf_logps_tiles(*{**dict(w=one, ldw=64, v=8, h=one, ldh=64, n=1, k=64, y=one, ig=-100, s=1.0, t=1,  # noqa: E731
                                                    p=one, tg=one, od=None, kp=None, ldk=0, l=one, lp=one, st=None), **k}.values())
    assert tiles(w=None) == tiles(v=0) == tiles(ldw=32) == tiles(s=0.0) == tiles(kp=one, ldk=64) == tiles(ldh=1 << 23) == 9001
    assert tiles(k=32) == tiles(w=72) == tiles(ldh=68) == tiles(kp=72, ldk=256) == 9007
    assert tiles(t=0) == 9003 and tiles(n=0) == 0
    none = (one, 0, 1.0, None, None, 0, None)
    assert hip.sf_logps_keep_grad(one, 256, 2, 1, 8, one, one, -100, one, one, 1, *none) == 9001
    assert hip.sf_logps_keep_grad(one, 264, 1, 1, 8, one, one, -100, one, one, 1, *none) == 9007
    assert hip.sf_logps_keep_grad(one, 256, 2, 2, 8, one, one, -100, one, one, 1, one, 1, 1.0, one, None, 0, None) == 9001
    assert hip.sf_logps_keep_grad(one, 256, 1, 1, 8, one, one, -100, one, one, 1, one, 1, 1.0, one, None, 1, None) == 9001
    grad = lambda **k: hip.sf_logps_hidden_grad(*{**dict(d=one, ld=32, n=1, w=one, ldw=8, v=8, h=8, by=one, s=None, t=1,  # noqa: E731
                                                         o=one, st=None), **k}.values())
    assert grad(n=0) == 0
    assert grad(d=None) == grad(w=None) == grad(by=None) == grad(o=None) == grad(v=0) == grad(h=0) == 9001
    assert grad(ld=31) == grad(ldw=7) == grad(n=1 << 31) == 9001 and grad(t=0) == grad(t=5) == 9003
    assert grad(ld=36) == grad(ldw=12) == grad(h=4) == 9007
    grad = lambda **k: hip.sf_logps_weight_grad(*{**dict(d=one, ld=8, n=64, v=8, h=one, k=8, s=None, t=1, o=one,  # noqa: E731
                                                         st=None), **k}.values())
    assert grad(d=None) == grad(h=None) == grad(o=None) == grad(v=0) == grad(k=0) == grad(n=0) == 9001
    assert grad(n=1 << 23) == grad(ld=7) == grad(k=1 << 23) == 9001 and grad(t=0) == 9003
    assert grad(n=65) == grad(ld=10) == grad(k=4) == grad(d=68) == grad(h=72) == grad(o=72) == 9007
    product = lambda **k: hip.sf_logps_hidden_product(*{**dict(d=one, ld=64, n=1, w=one, ldw=8, v=8, k=8, p=1,  # noqa: E731
                                                               o=one, t=1, st=None), **k}.values())
    assert product(n=0) == 0 and product(d=None) == product(w=None) == product(o=None) == product(v=0) == 9001
    assert product(k=0) == product(ld=56) == product(ldw=7) == product(p=0) == product(p=2) == product(n=1 << 31) == 9001
    assert product(v=512, ld=512, p=5) == 9001 and product(t=0) == 9003   # 8 steps: 2, 2, 2, 2 and none
    assert product(ld=68) == product(ldw=12) == product(k=4) == product(d=72) == product(o=72) == 9007
    rows = lambda h=one, ld=8, n=1, k=8, w=one, t=2, o=one: hip.sf_logps_weighted(h, ld, n, k, w, t, o, None)  # noqa: E731
    assert rows(n=0) == 0 and rows(h=None) == rows(w=None) == rows(o=None) == rows(k=0) == rows(ld=0) == 9001
    assert rows(t=0) == 9003 and rows(ld=12) == rows(k=4) == rows(h=72) == 9007
    assert hip.sf_logps_hidden(one, 8, 1, 8, None, 1, one, 64, None) == hip.sf_logps_hidden(one, 8, 1, 8, one, 1, one, 32, None) == 9001
    assert hip.sf_logps_sum(one, 3, 1, 8, one, 1, None, 0, None, 0, one, None, None) == 9001
    assert hip.sf_align_parts(0, 5) == 0 and hip.sf_align_parts(4, 100) == 4
    assert hip.sf_align_parts(4, 1 << 31) == 0 and hip.sf_align_parts(2, 1 << 20) == 2 * 512
    pref = lambda **k: hip.sf_pref_loss(*{**dict(lp=one, ld=8, ref=one, ldr=8, m=one, ldm=8, p=1, c=8, f=0, b=0.1, s=0.0,  # noqa: E731
                                                a=0, w=one, l=one, ch=one, r=one, co=None, st=None), **k}.values())
    assert pref(lp=None) == pref(c=0) == pref(p=0) == pref(ld=7) == pref(f=3) == pref(b=0.0) == pref(s=2.0) == 9001
    assert pref(w=8) == 9007
    pol = lambda **k: hip.sf_policy_loss(*{**dict(lp=one, ld=8, o=one, ldo=8, r=None, ldr=0, a=one, lda=8, t=1, m=one, ldm=8,  # noqa: E731
                                                  n=1, c=8, lo=-0.1, hi=0.1, k=0.0, s=0, w=one, l=one, kl=None, cl=one,
                                                  sl=None, we=None, st=None), **k}.values())
    assert pol(lp=None) == pol(n=0) == pol(lda=7) == pol(lo=0.5) == pol(hi=-1.0) == pol(r=one, ldr=8) == pol(kl=one) == 9001
    assert pol(w=24) == 9007
    assert hip.sf_pref_grad(one, one, one, 7, 1, 8, one, None) == hip.sf_policy_grad(one, None, one, 1, 8, one, None) == 9001
    assert hip.sf_act8_pack(None, 1, 8, one, 0, None) == hip.sf_act8_unpack(one, 5, 8, 4096, 1, None) == 9001


def test_ignored_tokens_may_hold_anything():
    g = torch.Generator().manual_seed(8)
    hidden, weight = torch.randn(6, 8, generator=g), torch.randn(20, 8, generator=g)
    labels = torch.tensor([1, -100, 3, -100, 5, 6])
    results = []
    for fill in (0.0, math.nan):
        h = hidden.clone()
        h[labels == -100] = fill
        h.requires_grad_(True)
        w = weight.clone().requires_grad_(True)
        lp = linear_logps(h, w, labels)
        results.append((lp.detach(), *torch.autograd.grad(lp.sum(), (h, w))))
    assert all(a.isfinite().all() and torch.equal(a, b) for a, b in zip(*results))


def test_parts_of_the_hidden_gradient():
    """Powers of two that the adding kernel takes, one where the tiles fill whole rounds."""
    from test1_amd.linear_logps import _hidden_parts

    class Weight:   # a weight without its memory
        def __init__(self, v, h):
            self.shape = torch.Size((v, h))

        def element_size(self):
            return 2

        def is_contiguous(self):
            return True

        def data_ptr(self):
            return 4096

    for (n, h, v), want in {(8190, 5120, 152_064): 2, (4092, 4096, 128_256): 1, (8190, 4096, 32_000): 1,
                            (8190, 2560, 50_257): 4, (3000, 5120, 32_000): 1, (4000, 3584, 152_064): 8,
                            (8190, 5120, 8192): 1}.items():
        assert _hidden_parts(n, Weight(v, h)) == want, (n, h, v)
    for n in range(256, 9000, 300):
        for h in (512, 896, 2048, 4096, 5120):
            for v in (5000, 16_384, 32_000, 152_064):
                p = _hidden_parts(n, Weight(v, h))
                assert p in (1, 2, 4, 8, 16) and (p == 1 or v // p >= 1024)


@pytest.mark.parametrize("bias", [False, True])
def test_token_logps_of_the_output_unit(bias):
    """log_softmax of the logits that the unit's forward gives, at the next labels."""
    from test1_amd.slide_fsdp import OutputLayer

    torch.manual_seed(0)
    unit = OutputLayer(torch.nn.LayerNorm(16), torch.nn.Linear(16, 50, bias=bias), 16)
    hidden = torch.randn(3, 9, 16, requires_grad=True)
    labels = torch.randint(0, 50, (3, 9))
    labels[1, 2:6] = -100
    got = unit.token_logps(hidden, labels, temperature=0.7)
    logits = unit(hidden)[1][:, :-1].double()
    want = torch.log_softmax(logits / 0.7, dim=-1).gather(-1, labels[:, 1:].clamp(min=0).unsqueeze(-1)).squeeze(-1)
    want = torch.where(labels[:, 1:] == -100, torch.zeros_like(want), want)
    assert got.shape == (3, 8) and got.dtype == torch.float32 and (got[1, 1:5] == 0).all()
    assert torch.allclose(got.double(), want, atol=2e-6)   # a few roundings of logits up to 5
    for a, b in zip(torch.autograd.grad(got.sum(), [hidden, *unit.lm_head.parameters()], retain_graph=True),
                    torch.autograd.grad(want.sum(), [hidden, *unit.lm_head.parameters()])):
        assert torch.allclose(a, b, atol=1e-4)
    labels[0, 3] = 50
    assert unit.token_logps(hidden, labels)[0, 2].isnan()


def test_what_an_objective_may_return():
    from collections import namedtuple

    from test1_amd.alignment import PreferenceLoss
    from test1_amd.slide_fsdp import _loss_of

    loss, other = torch.tensor(1.0), torch.tensor(2.0)
    for result in (loss, (loss, other), [loss, {}], (loss,), PreferenceLoss(loss, other, other),
                   namedtuple("Late", "metrics loss")(other, loss)):
        assert _loss_of(result) is loss
    for result in (None, 1.0, (), (1.0, loss), {"loss": loss}, namedtuple("Odd", "metrics loss")(other, 3.0)):
        with pytest.raises(TypeError, match="objective returns"):
            _loss_of(result)


def test_rows_of_the_backward():
    """All of them and kept up to 8 GiB, whole 64s otherwise, and never more hidden
    elements than the launch that transposes them takes."""
    from test1_amd.linear_logps import _backward_rows

    assert _backward_rows(4092, 128_256, 4096) == (4092, True)
    assert _backward_rows(40_000, 128_256, 4096) == (8320, False)
    assert _backward_rows(1 << 23, 128, 4096) == (1 << 23, True)
    assert _backward_rows((1 << 23) + 1, 128, 4096) == (1 << 22, False)   # 2 GiB of 256 words
    assert _backward_rows(10_000, 128_256, 1 << 22) == (8192, False)
    for n, v, h in ((1 << 24, 128, 4096), (40_000, 128_256, 1 << 22), (1 << 25, 64, 64), (100, 1 << 29, 64), (900, 64, 1 << 22)):
        rows, kept = _backward_rows(n, v, h)
        assert (rows == n if kept else rows % 64 == 0 or rows == n)
        assert -(-rows // 64) * (h // 64) <= 1 << 23, (n, v, h)
