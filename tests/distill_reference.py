"""Distillation in float64, a token at a time, with the bounds on an evaluation with
fp32 logits that the tests hold the kernels to."""

import math

import torch

from alignment_reference import HALF, U


def distill(hidden, weight, ids, logps, mask=None, scale=1.0, kind="forward", rest=True, grad=None):
    """(loss[, grad_hidden, grad_weight]) and their bounds.

    A logit is a sum of H products, wrong by at most 2 H U of the sum of magnitudes in
    any order, scaled once; a log-probability adds the softmax's own sums of up to
    512 terms in a row and a few roundings of its argument: e, the same for the
    logarithm of all other words' mass.  Every derivative by a logit is p times
    something of these; it is rounded to the inputs' type twice, relative to a
    token's largest, a weighted hidden row once more, a result once."""
    h, w = hidden.double(), weight.double()
    n, v = h.shape[0], w.shape[0]
    z = h @ w.t() * scale
    lse = torch.logsumexp(z, 1)
    logp = z - lse[:, None]
    ez = (h.abs() @ w.abs().t()).amax(1) * (2 * h.shape[1] + 2) * U * scale
    e = 2 * ez + (512 + 8 * (z.abs().amax(1) + lse.abs())) * U
    loss, eloss = torch.zeros(n, dtype=torch.float64, device=h.device), torch.zeros(n, dtype=torch.float64, device=h.device)
    dz, edz = torch.zeros_like(z), torch.zeros_like(z)
    biggest = torch.zeros_like(loss)
    half, tiny = HALF.get(hidden.dtype, (0.0, 0.0))
    for i in range(n):
        there = ~(logps[i] == -math.inf)
        if (mask is not None and not mask[i]) or not there.any():
            continue
        words, t = ids[i][there], logps[i][there].double()
        if ((words < 0) | (words >= v)).any() or words.unique().numel() < words.numel():
            loss[i], dz[i] = math.nan, math.nan
            continue
        lp = logp[i, words]
        others = torch.ones(v, dtype=torch.bool, device=h.device)
        others[words] = False
        outside = bool(others.any())
        if not rest:
            t = t - torch.logsumexp(t, 0)
        lp_rest = torch.logsumexp(logp[i][others], 0) if outside else torch.tensor(-math.inf, dtype=torch.float64, device=h.device)
        if rest and outside:
            q_rest = (1 - t.exp().sum()).clamp(min=2.0 ** -24 if kind == "reverse" else 0.0)
        else:
            q_rest = torch.zeros((), dtype=torch.float64, device=h.device)
        lp, t = torch.cat([lp, lp_rest.view(1)]), torch.cat([t, q_rest.log().view(1)])
        p, q = lp.exp(), t.exp()
        if kind == "forward":
            loss[i] = torch.where(q > 0, q * (t - lp), 0.0).sum()
            eloss[i] = q.sum() * e[i]
            slope, eslope = q.sum() * p - q, q.sum() * p * e[i]
        else:
            a = torch.where(p > 0, lp - t, 0.0)
            loss[i] = (p * a).sum()
            eloss[i] = e[i] * (p * (a.abs() + 1)).sum()
            slope = p * (a - loss[i])
            eslope = slope.abs() * e[i] + p * (e[i] + eloss[i])
        eloss[i] = 1.01 * eloss[i] + U * loss[i].abs()
        slope[-1] = slope[-1] if outside else 0.0
        biggest[i] = slope.abs().max()
        dz[i, words], edz[i, words] = slope[:-1], eslope[:-1]
        if outside:
            share = (logp[i][others] - lp_rest).exp()
            dz[i, others], edz[i, others] = share * slope[-1], share * (eslope[-1] + 2 * e[i] * slope[-1].abs())
    if grad is None:
        return (loss,), (eloss,)
    g = grad.double() * scale
    none = (g == 0) | ((loss == 0) & (biggest == 0))
    dz = torch.where(none[:, None], 0.0, dz * g[:, None])
    edz = edz * g.abs()[:, None] + dz.abs() * (2 * half + 8 * U)
    # fp16: relative to the largest row weight, half its least subnormal each time
    least = tiny * (2 * (g.abs() * biggest).max() if hidden.dtype == torch.float16 else 1.0)
    edz = edz + 2 * least
    h = torch.where(none[:, None], 0.0, h)
    gh, gw = dz @ w, dz.t() @ h
    egh = edz @ w.abs() + (dz.abs() @ w.abs()) * (2 * v * U) + half * gh.abs() + tiny
    egw = edz.t() @ h.abs() + (dz.abs().t() @ h.abs()) * (half + 2 * n * U) + half * gw.abs() + tiny
    if hidden.dtype == torch.float16:
        egw = egw + n * least
    return (loss, gh, gw), (eloss, egh * 1.01, egw * 1.01)
