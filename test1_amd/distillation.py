"""Distillation from a teacher's top log-probabilities under the output unit,
without keeping its [N, V] logits: each token's divergence of
``softmax(hidden @ weight.T / temperature)`` from what a teacher leaves of it
(``linear_top_logps``, ``sampling.top_logps``, ``SlideFSDP.top_logps``), with the
gradients of the hidden rows and of the weight.

The reference's output unit trains on labels alone (slide_fsdp.py:77-113).

Numerics: logits and the softmax's sums are fp32, as ``linear_logps``', the logits of
a token's likely words 64-bit; its few words, what lies outside them and the
divergence itself, a small difference of large terms, are in 64 bits.  Differences
of logits are taken before the temperature, however low it is.  The
gradient's products take 16-bit operands of 16-bit inputs: the derivatives by the
logits, rounded once (the exponentials that they come from are kept to 2^-10.5 of
themselves, in float16 2^-12.5), and the hidden rows as they are.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _native
from .fused_ce import _DTYPES, _PLAIN, _memory_is_value, _traced
from .linear_logps import _backward_rows, _chunk_rows, _f32_out, _hidden_parts, _label_kinds
from .sampling import TOP_MOST, TopLogps, top_logps

_FORMS = {"forward": _native.SF_DISTILL_FORWARD, "reverse": _native.SF_DISTILL_REVERSE}
_LEAST_REST = 2.0 ** -24


def _torch_distill(hidden, weight, ids, logps, mask, scale, kind, rest, bias=None):
    with torch.autocast(hidden.device.type, enabled=False):
        vocab = weight.shape[0]
        there = logps > -math.inf
        there = there | logps.isnan()
        _, at, outside = _label_kinds(ids, vocab, -1 - (1 << 62))
        order = torch.where(there, ids, -1).sort(dim=-1).values
        twice = (order[..., 1:] == order[..., :-1]) & (order[..., 1:] != -1)
        bad = (outside & there).any(dim=-1) | twice.any(dim=-1)
        taught = there.any(dim=-1)
        if mask is not None:
            taught = taught & mask
        bad = bad & taught
        there = there & (taught & ~bad).unsqueeze(-1)
        # what tokens without a loss hold does not reach the weight's gradient
        h = torch.where(taught.unsqueeze(-1), hidden, torch.zeros_like(hidden))
        logits = h.float() @ weight.float().t()
        if bias is not None:
            logits = logits + bias.float()
        logp = torch.log_softmax(logits.double() * scale, dim=-1)
        zero = torch.zeros((), dtype=torch.float64, device=hidden.device)
        lp = torch.where(there, logp.gather(-1, at), zero)
        t = torch.where(there, logps.double(), zero)
        q = torch.where(there, t.exp(), zero)
        named = q.sum(dim=-1, keepdim=True)
        if rest:
            # where a token's words are, or behind the vocabulary
            inside = torch.zeros((*logp.shape[:-1], vocab + 1), dtype=torch.bool, device=hidden.device)
            inside = inside.scatter(-1, torch.where(there, at, vocab), True)[..., :vocab]
            some = ~inside.all(dim=-1)
            others = torch.where(inside | ~some.unsqueeze(-1), -math.inf, logp)
            others = torch.where(some.unsqueeze(-1), others, zero)
            # relative to their largest, beside which the logarithm may be nothing: what they share comes of it
            largest = others.detach().amax(dim=-1, keepdim=True)
            largest = torch.where(largest.isfinite(), largest, zero)
            lp_rest = torch.where(some, (others - largest).exp().sum(dim=-1).log() + largest.squeeze(-1), zero)
            q_rest = (1 - named.squeeze(-1)).clamp(min=_LEAST_REST if kind == "reverse" else 0.0)
            q_rest = torch.where(some, q_rest, zero)
        else:
            t, q = t - named.log(), q / named
            some, lp_rest, q_rest = torch.zeros_like(taught), zero, torch.zeros_like(named.squeeze(-1))
        log_q_rest = torch.where(q_rest > 0, q_rest, 1.0).log()
        if kind == "forward":
            loss = torch.where(there & (q != 0), q * (t - lp), zero).sum(dim=-1)
            loss = loss + torch.where(q_rest > 0, q_rest * (log_q_rest - lp_rest), zero)
        else:
            loss = torch.where(there, lp.exp() * (lp - t), zero).sum(dim=-1)
            loss = loss + torch.where(some, lp_rest.exp() * (lp_rest - log_q_rest), zero)
        loss = torch.where(taught, torch.where(bad, logp[..., 0], loss), zero).float()
        return loss * torch.where(bad, math.nan, 1.0)


def _kernels_take(hidden, weight, ids, logps, mask) -> bool:
    given = (hidden, weight, ids, logps) if mask is None else (hidden, weight, ids, logps, mask)
    return (hidden.is_cuda and not _traced() and hidden.numel() > 0 and weight.shape[0] <= 1 << 30
            and ids.numel() // ids.shape[-1] < 1 << 31 and all(type(t) in _PLAIN and _memory_is_value(t) for t in given))


def _check_taught(shape, device, ids, logps, mask, temperature, kind, rest) -> None:
    """What a teacher leaves of ``shape`` tokens, and how it is to be taken."""
    if ids.shape != logps.shape or ids.dim() < 1 or ids.shape[:-1] != shape:
        raise ValueError("linear_distill: teacher_ids and teacher_logps of [..., K] expected, one row for each hidden row")
    if not 1 <= ids.shape[-1] <= TOP_MOST:
        raise ValueError(f"linear_distill: from 1 to {TOP_MOST} words of each token expected, got {ids.shape[-1]}")
    if ids.dtype != torch.int64 or logps.dtype != torch.float32:
        raise TypeError(f"linear_distill: int64 ids and float32 log-probabilities expected, got {ids.dtype}, {logps.dtype}")
    if mask is not None and mask.dtype != torch.bool:
        raise TypeError(f"linear_distill: a bool mask expected, got {mask.dtype}")
    if mask is not None and mask.shape != shape:
        raise ValueError(f"linear_distill: the mask has to be {tuple(shape)}")
    if any(t is not None and t.device != device for t in (ids, logps, mask)):
        raise ValueError("linear_distill: all tensors have to be on one device")
    if not 1e-30 <= temperature <= 1e30:   # neither it nor its inverse leaves fp32
        raise ValueError(f"linear_distill: a temperature above 0, from 1e-30 to 1e30, expected, got {temperature}")
    if kind not in _FORMS:
        raise ValueError(f"linear_distill: kind must be one of {sorted(_FORMS)}, got {kind!r}")
    if kind == "reverse" and not rest:
        raise ValueError("linear_distill: kind 'reverse' needs the rest: a student's words outside the teacher's have no q")
    if logps.requires_grad and torch.is_grad_enabled():
        raise ValueError("linear_distill: teacher_logps takes no gradient; detach it")


def linear_distill(hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor, teacher_logps: torch.Tensor,
                   mask: Optional[torch.Tensor] = None, temperature: float = 1.0, kind: str = "forward",
                   rest: bool = True) -> torch.Tensor:
    """Each token's divergence of p = ``softmax(hidden @ weight.T /
    temperature)`` from a teacher's probabilities of a few words, float32, of
    ``mask``'s shape.

    ``hidden`` [..., H] and ``weight`` [V, H] of one float type (bfloat16,
    float16 or float32); ``teacher_ids`` [..., K] int64 and ``teacher_logps``
    [..., K] float32, K up to ``TOP_MOST`` (128): what ``top_logps`` gives, at
    the same temperature, in any order; a log-probability of -infinity stands
    for no word, whatever its id.  ``mask`` [...] bool: the tokens that count.

    With q the teacher's probabilities:

    * ``"forward"``: sum of q (log q - log p)
    * ``"reverse"``: sum of p (log p - log q)

    over the teacher's words and, as one outcome, all others (``rest``), which
    have 1 - sum q, in ``"reverse"`` at least 2^-24.  ``rest=False``
    (``"forward"``): over the words alone, q divided by its sum.

    0, without gradient, where the mask is False or the teacher has no word; NaN
    where an id is outside the vocabulary or stands twice.  Differentiable once by
    ``hidden`` and ``weight``; on a GPU, tokens whose upstream gradient is 0 leave the
    gradients alone, whatever their hidden states hold.  Under ``no_grad`` nothing is kept.  Autocast does not change
    it.  It is not multiplied by temperature^2."""
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError("linear_distill: hidden [..., H] and weight [V, H] expected")
    if hidden.dtype not in _DTYPES or weight.dtype != hidden.dtype:
        raise TypeError(f"linear_distill: hidden and weight of one float type expected, got {hidden.dtype}, {weight.dtype}")
    if weight.device != hidden.device:
        raise ValueError("linear_distill: all tensors have to be on one device")
    if weight.shape[0] == 0:
        raise ValueError("linear_distill: an empty vocabulary")
    _check_taught(hidden.shape[:-1], hidden.device, teacher_ids, teacher_logps, mask, temperature, kind, rest)
    scale = 1.0 / float(temperature)
    if not _kernels_take(hidden, weight, teacher_ids, teacher_logps, mask):
        return _torch_distill(hidden, weight, teacher_ids, teacher_logps, mask, scale, kind, rest)
    rows = hidden.reshape(-1, hidden.shape[-1])
    ids, logps = (t.reshape(-1, t.shape[-1]) for t in (teacher_ids, teacher_logps))
    flat = None if mask is None else mask.reshape(-1)
    step, keep, nparts = rows.shape[0], False, 1
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        step, keep = _backward_rows(step, *weight.shape)
        nparts = _hidden_parts(step, weight)
    loss = _native.ops().linear_distill(rows, weight, ids, logps, flat, _FORMS[kind], bool(rest), scale, nparts, step, keep)
    if loss is None:
        return _torch_distill(hidden, weight, teacher_ids, teacher_logps, mask, scale, kind, rest)
    return loss.view(hidden.shape[:-1])


# ---------------------------------------------------------------------------
def _logits32(hidden: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``hidden @ weight.T + bias`` of a few rows, not rounded to 16 bits in between."""
    if hidden.is_cuda and hidden.dim() == 2 and hidden.numel() > 0 and type(hidden) in _PLAIN and not _traced():
        z = torch.mm(hidden, weight.t(), **_f32_out(hidden.dtype))
    else:
        z = hidden.float() @ weight.float().t()
    return z if bias is None else z.add_(bias)


@torch.no_grad()
def linear_top_logps(hidden: torch.Tensor, weight: torch.Tensor, k: int, temperature: float = 1.0,
                     bias: Optional[torch.Tensor] = None) -> TopLogps:
    """``top_logps`` of ``hidden @ weight.T + bias``, whose logits are fp32 and
    made 1 GiB at a time.  ``hidden`` [..., H] and ``weight`` [V, H] of one
    float type, ``bias`` [V] or None.  No gradient."""
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError("linear_top_logps: hidden [..., H] and weight [V, H] expected")
    if hidden.dtype not in _DTYPES or weight.dtype != hidden.dtype:
        raise TypeError(f"linear_top_logps: hidden and weight of one float type expected, got {hidden.dtype}, {weight.dtype}")
    if weight.device != hidden.device or (bias is not None and bias.device != hidden.device):
        raise ValueError("linear_top_logps: all tensors have to be on one device")
    if weight.shape[0] == 0 or (bias is not None and bias.shape != weight.shape[:1]):
        raise ValueError(f"linear_top_logps: a vocabulary and a bias of it expected, got {tuple(weight.shape)}")
    rows = hidden.reshape(-1, hidden.shape[-1])
    step = _chunk_rows(weight.shape[0])
    with torch.autocast(hidden.device.type, enabled=False):
        parts = [top_logps(_logits32(rows[s:s + step], weight, bias), k, temperature)
                 for s in range(0, max(1, rows.shape[0]), step)]
    logps, ids = (torch.cat(t) if len(parts) > 1 else t[0] for t in zip(*parts))
    return TopLogps(logps.view(*hidden.shape[:-1], k), ids.view(*hidden.shape[:-1], k))
