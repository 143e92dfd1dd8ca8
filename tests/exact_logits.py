"""Distillation where every logit is a small whole number: products of 16-bit or fp32
operands hold them exactly, whatever order their terms are added in, so that a low
temperature's large differences are known exactly too."""

import math

import torch

from alignment_reference import HALF, U


def inputs(shape, dtype, dev, seed=0):
    """hidden, weight, ids, logps of a teacher of its own, mask, upstream."""
    n, h, v, k = shape
    g = torch.Generator(device=dev).manual_seed(seed + n + h + v)
    hidden = torch.randint(-2, 3, (n, h), generator=g, device=dev).to(dtype)
    weight = torch.randint(-2, 3, (v, h), generator=g, device=dev).to(dtype)
    ids = torch.rand(n, v, generator=g, device=dev).argsort(dim=1)[:, :k].contiguous()
    logps = torch.log_softmax(torch.randn(n, v, generator=g, device=dev) * 2, dim=1).gather(1, ids) - 0.1
    # some teachers name the student's largest words
    ids[::3] = (hidden[::3].double() @ weight.double().t()).topk(k, dim=1).indices
    mask = torch.rand(n, generator=g, device=dev) < 0.85
    mask[0] = True
    return hidden, weight, ids, logps, mask, torch.randn(n, generator=g, device=dev)


def distill(hidden, weight, ids, logps, mask, temperature, kind, rest, grad):
    """(loss, grad_hidden, grad_weight) in float64 and the bounds of the kernels'.

    All differences of logits are exact.  The mass of the words outside a token's
    own is a sum in fp32, of 512 terms in a row at most, each within 8 U: e.  The
    words' own terms are in 64 bits.  A derivative by a logit is a token's over its
    largest one, the largest one, their product with the upstream and the scale: 8
    roundings; of other words also an exponential of up to 32 octaves' exponent, off by
    40 U, and of 16-bit operands kept to 16 bits of its logarithm, off by half a type's rounding at
    most; rounded to that type before the products, whose sums of n or v terms are in
    fp32, and after."""
    h, w = hidden.double(), weight.double()
    n, v = h.shape[0], w.shape[0]
    scale, e = 1.0 / temperature, 520 * U
    z = h @ w.t()
    zero = torch.zeros(n, dtype=torch.float64, device=h.device)
    loss, eloss, dz, edz, biggest = zero.clone(), zero.clone(), torch.zeros_like(z), torch.zeros_like(z), zero.clone()
    for i in range(n):
        if not mask[i]:
            continue
        named = torch.zeros(v, dtype=torch.bool, device=h.device)
        named[ids[i]] = True
        d = (z[i] - z[i].max()) * scale
        lse = torch.logsumexp(d, 0)
        top = d[~named].max()
        within = torch.logsumexp(d[~named] - top, 0)
        t = logps[i].double()
        if not rest:
            t = t - torch.logsumexp(t, 0)
        least = 2.0 ** -24 if kind == "reverse" else 0.0
        left = (1 - t.exp().sum()).clamp(min=least) if rest else torch.zeros((), dtype=torch.float64, device=h.device)
        lp, t = torch.cat([d[ids[i]] - lse, (top + within - lse).view(1)]), torch.cat([t, left.log().view(1)])
        p, q = lp.exp(), t.exp()
        if kind == "forward":
            loss[i] = torch.where(q > 0, q * (t - lp), 0.0).sum()
            slope = q.sum() * p - q
            eloss[i], eslope = q.sum() * e, q.sum() * p * e
        else:
            a = torch.where(p > 0, lp - t, 0.0)
            loss[i] = (p * a).sum()
            slope = p * (a - loss[i])
            eloss[i] = e * (p * (a.abs() + 1)).sum()
            eslope = slope.abs() * e + p * (e + eloss[i])
        # in 64 bits |loss| / T cancels among larger terms
        eloss[i] += U * loss[i].abs() + 2.0 ** -50 * (1 + torch.where(q > 0, q * lp.abs(), 0.0).sum())
        biggest[i] = slope.abs().max()
        share = (d[~named] - top - within).exp()
        dz[i, ids[i]], edz[i, ids[i]] = slope[:-1], eslope[:-1]
        dz[i, ~named], edz[i, ~named] = share * slope[-1], share * (eslope[-1] + (e + 40 * U) * slope[-1].abs())
    half, tiny = HALF.get(hidden.dtype)
    half = half if hidden.dtype != torch.float32 else 0.0
    g = grad.double() * scale
    dz, edz = dz * g[:, None], edz * g.abs()[:, None]
    edz = edz + dz.abs() * (2 * half + 8 * U)
    # D is held over c, the largest derivative times its upstream: half a least subnormal of D is c halves
    # of one here, up to 2 c after the division's and the power of two's own roundings
    c = (g.abs() * biggest).max()
    least = tiny * (2 * c if hidden.dtype == torch.float16 else max(1.0, 2 * c))
    edz = edz + 2 * least
    gh, gw = dz @ w, dz.t() @ h
    half, tiny = HALF[hidden.dtype]
    egh = edz @ w.abs() + (dz.abs() @ w.abs()) * (2 * v * U) + half * gh.abs() + tiny
    egw = edz.t() @ h.abs() + (dz.abs().t() @ h.abs()) * (2 * n * U) + half * gw.abs() + tiny
    return (loss, gh, gw), (eloss, egh * 1.01, egw * 1.01)
