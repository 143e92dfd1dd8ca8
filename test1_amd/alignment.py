"""Losses over token log-probabilities, for fine-tuning by preferences or by
rewards: the preference loss of paired sequences and the clipped policy loss
with a KL term, each with its gradient.

The reference trains on cross entropy alone (slide_fsdp.py:85-113); these are
objectives beside it.  ``linear_logps`` gives the log-probabilities they take,
``SlideFSDP.forward(..., objective=...)`` runs a step on them.

The kernels (``csrc/sf_align.hip``) read every token once and write its
gradient once.  On a host, and for calls that the kernels cannot serve (traced,
batched by vmap, forward-mode derivatives), the same formulas run as torch
operations, differentiable as those are; the kernels' gradients are not
differentiated again.  Masked tokens count for nothing, whatever stands there.
"""

from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .fused_ce import _PLAIN, _memory_is_value, _saved_plain, _traced

_FORMS = {"sigmoid": _native.SF_PREF_SIGMOID, "hinge": _native.SF_PREF_HINGE, "ipo": _native.SF_PREF_IPO}
_REDUCTIONS = ("token", "sequence")


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor               # scalar, differentiable by the log-probabilities
    chosen_rewards: torch.Tensor     # [P] beta times the log ratio of each chosen sequence
    rejected_rewards: torch.Tensor   # [P]


class PolicyLoss(NamedTuple):
    loss: torch.Tensor               # scalar, differentiable by the log-probabilities
    kl: Optional[torch.Tensor]       # scalar mean of exp(q) - 1 - q; None without ref_logps
    clip_fraction: torch.Tensor      # scalar mean of the tokens that were clipped


def _check_tokens(what: str, logps: torch.Tensor, mask: torch.Tensor, **others: Optional[torch.Tensor]) -> None:
    if logps.dim() != 2:
        raise ValueError(f"{what}: log-probabilities of [rows, tokens] expected, got {tuple(logps.shape)}")
    if mask.dtype != torch.bool:
        raise TypeError(f"{what}: a bool mask expected, got {mask.dtype}")
    if logps.dtype != torch.float32:
        raise TypeError(f"{what}: float32 log-probabilities expected, got {logps.dtype}")
    if mask.shape != logps.shape or mask.device != logps.device:
        raise ValueError(f"{what}: the mask has to be {tuple(logps.shape)} on {logps.device}")
    for name, t in others.items():
        if t is None:
            continue
        if t.dtype != torch.float32:
            raise TypeError(f"{what}: float32 {name} expected, got {t.dtype}")
        if t.device != logps.device:
            raise ValueError(f"{what}: {name} has to be on {logps.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what}: {name} takes no gradient; detach it")


def _kernels_take(logps: torch.Tensor, *others: Optional[torch.Tensor]) -> bool:
    if not logps.is_cuda or logps.numel() == 0 or _traced():
        return False
    return all(t is None or (type(t) in _PLAIN and _memory_is_value(t)) for t in (logps, *others))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernels read it: the elements of a row side by side, rows
    any whole number of elements apart that holds one."""
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        return t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


@functools.lru_cache(maxsize=256)
def _parts(rows: int, cols: int) -> int:
    return _native.hip().sf_align_parts(rows, cols)


def _stream() -> int:
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


class _on_device:
    """The tensors' device as the current one, without cost where it is."""

    def __new__(cls, t: torch.Tensor):
        return _HERE if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


class _Nothing:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_HERE = _Nothing()


# ---------------------------------------------------------------------------
def _pref_kernels(logps, ref, mask, form, beta, smoothing, average, need_grad):
    rows, cols = logps.shape
    pairs = rows // 2
    logps, ref = _rows(logps), _rows(ref)
    dev = logps.device
    parts = torch.empty(2 * _parts(rows, cols), dtype=torch.float64, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    chosen = torch.empty(pairs, dtype=torch.float32, device=dev)
    rejected = torch.empty(pairs, dtype=torch.float32, device=dev)
    coef = torch.empty(rows, dtype=torch.float32, device=dev) if need_grad else None
    _native.check(_native.hip().sf_pref_loss(
        logps.data_ptr(), _ld(logps), ref.data_ptr(), _ld(ref), mask.data_ptr(), _ld(mask), pairs, cols, form, beta,
        smoothing, average, parts.data_ptr(), loss.data_ptr(), chosen.data_ptr(), rejected.data_ptr(),
        coef.data_ptr() if need_grad else None, _stream()), "sf_pref_loss")
    return loss, chosen, rejected, coef


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, ref, mask, form, beta, smoothing, average):
        ctx.set_materialize_grads(False)
        loss, chosen, rejected, coef = _pref_kernels(logps, ref, mask, form, beta, smoothing, average, True)
        ctx.save_for_backward(coef, mask)
        ctx.mark_non_differentiable(chosen, rejected)
        return loss, chosen, rejected

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, *_):
        if grad_loss is None:
            return (None,) * 7
        coef, mask = ctx.saved_tensors
        if (not _traced() and _saved_plain(coef, torch.float32, grad_loss.device) and type(mask) is torch.Tensor
                and mask.dtype == torch.bool and mask.device == coef.device and _rows(mask) is mask
                and _plain_grad(grad_loss)):
            with _on_device(coef):
                rows, cols = mask.shape
                grad = torch.empty((rows, cols), dtype=torch.float32, device=coef.device)
                _native.check(_native.hip().sf_pref_grad(grad_loss.data_ptr(), coef.data_ptr(), mask.data_ptr(),
                                                         _ld(mask), rows, cols, grad.data_ptr(), _stream()),
                              "sf_pref_grad")
        else:
            coef = coef.to(torch.float32) * grad_loss
            grad = torch.where(mask.to(torch.bool), coef.unsqueeze(1), torch.zeros((), device=coef.device))
        return grad, None, None, None, None, None, None


def _plain_grad(g: torch.Tensor) -> bool:
    return type(g) is torch.Tensor and g.is_cuda and g.dtype == torch.float32 and g.numel() == 1 and _memory_is_value(g)


def _log_sigmoid(x: torch.Tensor) -> torch.Tensor:
    return torch.nn.functional.logsigmoid(x)


def _pref_torch(logps, ref, mask, kind, beta, smoothing, average):
    ratio = torch.where(mask, logps - ref, torch.zeros_like(logps)).sum(dim=1)
    if average:
        ratio = ratio / mask.sum(dim=1).clamp(min=1)
    chosen, rejected = ratio.chunk(2)
    gap = chosen - rejected
    if kind == "sigmoid":
        terms = 0.0
        if smoothing < 1:
            terms = terms - (1 - smoothing) * _log_sigmoid(beta * gap)
        if smoothing > 0:
            terms = terms - smoothing * _log_sigmoid(-beta * gap)
    elif kind == "hinge":
        terms = torch.relu(1 - beta * gap)
    else:
        terms = (gap - 1 / (2 * beta)).square()
    return PreferenceLoss(terms.mean(), (beta * chosen).detach(), (beta * rejected).detach())


def preference_loss(logps: torch.Tensor, ref_logps: torch.Tensor, mask: torch.Tensor, beta: float = 0.1,
                    kind: str = "sigmoid", label_smoothing: float = 0.0, average: bool = False) -> PreferenceLoss:
    """Preference loss of P pairs of sequences.

    ``logps`` [2 P, T] float32: the policy's log-probabilities of the tokens,
    rows 0 to P - 1 the chosen sequences, rows P to 2 P - 1 the rejected ones
    in the same order; ``ref_logps`` the reference policy's; ``mask`` bool, the
    tokens that count.  With R the sum of a row's ``logps - ref_logps``
    (``average``: its mean) and D the chosen R less the rejected, the loss is
    the mean over the pairs of

    * ``"sigmoid"``: -(1 - s) log sigmoid(beta D) - s log sigmoid(-beta D),
      s = ``label_smoothing``
    * ``"hinge"``: max(0, 1 - beta D)
    * ``"ipo"``: (D - 1 / (2 beta))^2

    A row without tokens has R = 0."""
    _check_tokens("preference_loss", logps, mask, ref_logps=ref_logps)
    if ref_logps.shape != logps.shape:
        raise ValueError(f"preference_loss: ref_logps has to be {tuple(logps.shape)}")
    if logps.shape[0] == 0 or logps.shape[0] % 2:
        raise ValueError(f"preference_loss: an even number of rows expected, chosen then rejected, got {logps.shape[0]}")
    if kind not in _FORMS:
        raise ValueError(f"preference_loss: kind must be one of {sorted(_FORMS)}, got {kind!r}")
    if not (beta > 0 and math.isfinite(beta)):
        raise ValueError("preference_loss: beta must be above 0")
    if not 0 <= label_smoothing <= 1 or (label_smoothing and kind != "sigmoid"):
        raise ValueError("preference_loss: label_smoothing is in [0, 1], for kind 'sigmoid'")
    if not _kernels_take(logps, ref_logps, mask):
        return _pref_torch(logps, ref_logps, mask, kind, beta, label_smoothing, average)
    args = (_FORMS[kind], float(beta), float(label_smoothing), bool(average))
    with _on_device(logps):
        mask = _rows(mask)
        if torch.is_grad_enabled() and logps.requires_grad:
            return PreferenceLoss(*_Preference.apply(logps, ref_logps, mask, *args))
        return PreferenceLoss(*_pref_kernels(logps, ref_logps, mask, *args, False)[:3])


# ---------------------------------------------------------------------------
def _policy_kernels(logps, old, adv, mask, ref, log_low, log_high, kl_coef, sequences, need_grad):
    rows, cols = logps.shape
    logps, old, mask = _rows(logps), _rows(old), _rows(mask)
    per_token = adv.dim() == 2
    if per_token:
        adv = _rows(adv)
    if ref is not None:
        ref = _rows(ref)
    dev = logps.device
    parts = torch.empty(4 * _parts(rows, cols), dtype=torch.float64, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    kl = torch.empty((), dtype=torch.float32, device=dev) if ref is not None else None
    clipped = torch.empty((), dtype=torch.float32, device=dev)
    slope = torch.empty((rows, cols), dtype=torch.float32, device=dev) if need_grad else None
    weight = torch.empty(rows, dtype=torch.float32, device=dev) if need_grad else None
    _native.check(_native.hip().sf_policy_loss(
        logps.data_ptr(), _ld(logps), old.data_ptr(), _ld(old), None if ref is None else ref.data_ptr(),
        0 if ref is None else _ld(ref), adv.data_ptr(), _ld(adv) if per_token else adv.stride(0), per_token,
        mask.data_ptr(), _ld(mask), rows, cols, log_low, log_high, kl_coef, sequences, parts.data_ptr(),
        loss.data_ptr(), None if kl is None else kl.data_ptr(), clipped.data_ptr(),
        slope.data_ptr() if need_grad else None, weight.data_ptr() if need_grad else None, _stream()), "sf_policy_loss")
    return loss, kl, clipped, slope, weight


class _Policy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, *args):
        ctx.set_materialize_grads(False)
        loss, kl, clipped, slope, weight = _policy_kernels(logps, *args, True)
        ctx.save_for_backward(slope, weight)
        ctx.mark_non_differentiable(*(t for t in (kl, clipped) if t is not None))
        return loss, kl, clipped

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, *_):
        if grad_loss is None:
            return (None,) * 9
        slope, weight = ctx.saved_tensors
        dev = grad_loss.device
        if (not _traced() and _saved_plain(slope, torch.float32, dev) and _saved_plain(weight, torch.float32, dev)
                and _plain_grad(grad_loss)):
            with _on_device(slope):
                rows, cols = slope.shape
                grad = torch.empty_like(slope)
                _native.check(_native.hip().sf_policy_grad(grad_loss.data_ptr(), weight.data_ptr(), slope.data_ptr(),
                                                           rows, cols, grad.data_ptr(), _stream()), "sf_policy_grad")
        else:
            grad = slope.to(torch.float32) * (weight.to(torch.float32) * grad_loss).unsqueeze(-1)
        return (grad,) + (None,) * 8


def _mean_torch(x, mask, sequences):
    x = torch.where(mask, x, torch.zeros_like(x))
    if not sequences:
        return x.sum() / mask.sum()
    count = mask.sum(dim=1)
    return (x.sum(dim=1) / count.clamp(min=1)).sum() / (count > 0).sum()


def _policy_torch(logps, old, adv, mask, ref, log_low, log_high, kl_coef, sequences):
    adv = adv if adv.dim() == 2 else adv.unsqueeze(1).expand_as(logps)
    # masked tokens leave before the exponentials, whose gradients would be NaN
    zero = torch.zeros_like(logps)
    d = torch.where(mask, logps - old, zero)
    adv = torch.where(mask, adv, zero)
    clipped = torch.where(adv > 0, d > log_high, (adv < 0) & (d < log_low))
    terms = -torch.where(clipped, d.clamp(log_low, log_high), d).exp() * adv
    kl = None
    if ref is not None:
        q = torch.where(mask, ref - logps, zero)
        each = torch.expm1(q) - q
        terms = terms + kl_coef * each
        kl = _mean_torch(each.detach(), mask, sequences)
    return PolicyLoss(_mean_torch(terms, mask, sequences), kl,
                      _mean_torch(clipped.to(torch.float32), mask, sequences))


def policy_loss(logps: torch.Tensor, old_logps: torch.Tensor, advantages: torch.Tensor, mask: torch.Tensor,
                ref_logps: Optional[torch.Tensor] = None, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0, reduction: str = "token") -> PolicyLoss:
    """Clipped policy loss, with a KL term towards a reference policy if
    ``ref_logps`` is given.

    ``logps`` [B, T] float32: the policy's log-probabilities of the sampled
    tokens; ``old_logps`` those of the policy that sampled them;
    ``advantages`` [B, T], or [B]: one for all tokens of a row; ``mask`` bool,
    the tokens that count.  With d = logps - old_logps and q = ref_logps -
    logps a token's term is

        -min(exp(d) A, clip(exp(d), 1 - clip_low, 1 + clip_high) A)
            + kl_coef (exp(q) - 1 - q)

    Whether a token is clipped is decided on d, against log(1 - clip_low) and
    log(1 + clip_high) in float32.  ``reduction``: ``"token"``, the mean over
    all tokens, or ``"sequence"``, the mean over the rows with any of their own
    means.  Without any token the means are NaN and the gradient 0."""
    _check_tokens("policy_loss", logps, mask, old_logps=old_logps, advantages=advantages, ref_logps=ref_logps)
    for name, t in (("old_logps", old_logps), ("ref_logps", ref_logps)):
        if t is not None and t.shape != logps.shape:
            raise ValueError(f"policy_loss: {name} has to be {tuple(logps.shape)}")
    if advantages.shape != logps.shape and advantages.shape != logps.shape[:1]:
        raise ValueError(f"policy_loss: advantages have to be {tuple(logps.shape)} or {tuple(logps.shape[:1])}")
    if not (0 <= clip_low <= 1 and clip_high >= 0):
        raise ValueError("policy_loss: clip_low in [0, 1] and clip_high from 0 expected")
    if not math.isfinite(kl_coef):
        raise ValueError("policy_loss: a finite kl_coef expected")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"policy_loss: reduction must be one of {_REDUCTIONS}, got {reduction!r}")
    log_low = math.log1p(-clip_low) if clip_low < 1 else -math.inf
    args = (old_logps, advantages, mask, ref_logps, log_low, math.log1p(clip_high), float(kl_coef),
            reduction == "sequence")
    if not _kernels_take(logps, old_logps, advantages, mask, ref_logps):
        return _policy_torch(logps, *args)
    with _on_device(logps):
        if torch.is_grad_enabled() and logps.requires_grad:
            return PolicyLoss(*_Policy.apply(logps, *args))
        return PolicyLoss(*_policy_kernels(logps, *args, False)[:3])
