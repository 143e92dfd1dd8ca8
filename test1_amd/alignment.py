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

import math
from typing import NamedTuple, Optional

import torch

from . import _native
from .fused_ce import _traced

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
    if logps.is_cuda and logps.numel() > 0 and not _traced():
        out = _native.ops().pref_loss(logps, ref_logps, mask, _FORMS[kind], beta, label_smoothing, average)
        if out is not None:
            return PreferenceLoss(*out)
    return _pref_torch(logps, ref_logps, mask, kind, beta, label_smoothing, average)


# ---------------------------------------------------------------------------
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
    if logps.is_cuda and logps.numel() > 0 and not _traced():
        out = _native.ops().policy_loss(logps, *args)
        if out is not None:
            return PolicyLoss(*out)
    return _policy_torch(logps, *args)
