"""Plain 64-bit forms of the losses over token log-probabilities, the token
log-probabilities themselves and the 8-bit checkpoints, with the bounds on a
32-bit evaluation that the tests hold the kernels to."""

import math

import torch

U = 2.0 ** -24   # unit roundoff of float32
# unit roundoff and half the least subnormal of each type
HALF = {torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25),
        torch.float32: (2.0 ** -24, 2.0 ** -150)}


def preference(lp, ref, mask, beta, kind, smoothing, average):
    """(loss, chosen, rejected, grad) and the bounds of a 32-bit evaluation of
    each.  A row's sum: one rounding of each difference, at most four terms
    added in 32 bits, the rest in 64: 4 U of the sum of magnitudes."""
    d = torch.where(mask, lp.double() - ref.double(), torch.zeros(lp.shape, dtype=torch.float64, device=lp.device))
    r, er = d.sum(1), 4 * U * d.abs().sum(1)
    w = 1 / mask.sum(1).clamp(min=1).double() if average else torch.ones_like(r)
    r, er = r * w, er * w
    p = r.numel() // 2
    gap, egap = r[:p] - r[p:], er[:p] + er[p:]
    x = beta * gap
    if kind == "sigmoid":
        sp = torch.nn.functional.softplus
        terms = (1 - smoothing) * sp(-x) + smoothing * sp(x)
        slope = beta * (smoothing * torch.sigmoid(x) - (1 - smoothing) * torch.sigmoid(-x))
        eterm, eslope = beta * egap, beta * beta / 4 * egap
    elif kind == "hinge":
        terms, slope = torch.relu(1 - x), -beta * (x < 1).double()
        eterm, eslope = beta * egap, 0 * egap
        assert ((x - 1).abs() > beta * egap).all(), "a pair at the corner: take another seed"
    else:
        off = gap - 0.5 / beta
        terms, slope = off * off, 2 * off
        eterm, eslope = 2 * off.abs() * egap + egap * egap, 2 * egap
    grad = torch.cat([slope, -slope]) * w / p
    egrad = torch.cat([eslope, eslope]) * w / p + 4 * U * grad.abs()
    m = mask.double()
    return ((terms.mean(), beta * r[:p], beta * r[p:], grad[:, None] * m),
            (eterm.mean() + 2 * U * terms.mean().abs(), beta * er[:p] + 2 * U * (beta * r[:p]).abs(),
             beta * er[p:] + 2 * U * (beta * r[p:]).abs(), egrad[:, None] * m))


def policy(lp, old, adv, mask, ref, low, high, kl_coef, reduction):
    """(loss, kl, clip_fraction, grad) and the bounds of a 32-bit evaluation.
    A token's exponentials: their argument is rounded once, they are within 2
    ulp (4 U); a product and a sum more, and up to four tokens added."""
    zero = torch.zeros(lp.shape, dtype=torch.float64, device=lp.device)
    adv = adv if adv.dim() == 2 else adv[:, None].expand(lp.shape)
    a = torch.where(mask, adv.double(), zero)
    d32 = lp - old   # the decision is on the 32-bit difference
    lo = torch.tensor(math.log1p(-low) if low < 1 else -math.inf, dtype=torch.float32, device=lp.device)
    hi = torch.tensor(math.log1p(high), dtype=torch.float32, device=lp.device)
    clipped = mask & (((adv > 0) & (d32 > hi)) | ((adv < 0) & (d32 < lo)))
    d = torch.where(mask, lp.double() - old.double(), zero)
    dc = torch.where(clipped, torch.where(a > 0, hi.double(), lo.double()), d)
    ra = dc.exp() * a
    terms, slope = -ra, torch.where(clipped, zero, -ra)
    era = ra.abs() * (dc.abs() + 10) * U
    eterm, eslope = era.clone(), era.clone()
    each = eeach = zero
    if ref is not None:
        q = torch.where(mask, ref.double() - lp.double(), zero)
        em1 = torch.expm1(q)
        each = em1 - q
        eem1 = (q.abs() * q.exp() + 4 * em1.abs()) * U
        # beyond 1/2 a difference of em1 and q, below a series of nine terms
        eeach = torch.where(q.abs() > 0.5, eem1 + (q.abs() + each) * U, em1.abs() * q.abs() * U + 24 * each * U)
        terms = terms + kl_coef * each
        slope = slope - kl_coef * em1
        eterm = eterm + abs(kl_coef) * (eeach + 4 * each * U) + 4 * terms.abs() * U
        eslope = eslope + abs(kl_coef) * (eem1 + 4 * em1.abs() * U) + 4 * slope.abs() * U
    m = mask.double()
    if reduction == "token":
        w = m / m.sum()
    else:
        n = m.sum(1, keepdim=True)
        w = m / n.clamp(min=1) / (n > 0).sum()
    w = torch.where(mask, w, zero)
    none = not bool(mask.any())
    nan = torch.tensor(math.nan, dtype=torch.float64, device=lp.device)
    # terms of a lane are added four at a time in 32 bits
    total = lambda x, ex: nan if none else (x * w).sum()  # noqa: E731
    bound = lambda x, ex: ((ex + 4 * U * x.abs()) * w).sum() + 2 * U * (x * w).sum().abs()  # noqa: E731
    c = clipped.double()
    return ((total(terms, eterm), total(each, eeach), total(c, zero), slope * w),
            (bound(terms, eterm), bound(each, eeach), bound(c, zero), (eslope + 6 * U * slope.abs()) * w))


def logps(hidden, weight, labels, scale=1.0, ignore_index=-100, grad=None):
    """(logp[, grad_hidden, grad_weight]) in 64 bits and the bounds of an
    evaluation with fp32 logits: each logit is a sum of K products, wrong by at
    most 2 K U of the sum of magnitudes in any order, scaled once; the softmax
    adds up to 512 terms in a row and takes a few roundings of its argument.
    An element of the logits' gradient is rounded to the inputs' type twice, a
    weighted hidden row once more, a result once."""
    h, w = hidden.double(), weight.double()
    z = h @ w.t() * scale
    ez = (h.abs() @ w.abs().t()).amax(1) * (2 * h.shape[1] + 2) * U * scale
    ys = labels.clamp(0, w.shape[0] - 1)
    rows = torch.arange(len(labels), device=h.device)
    lse = torch.logsumexp(z, 1)
    lp = z[rows, ys] - lse
    big = z.abs().amax(1) + lse.abs()
    ignored, bad = labels == ignore_index, (labels != ignore_index) & ((labels < 0) | (labels >= w.shape[0]))
    lp[ignored] = 0.0
    lp[bad] = math.nan
    e = torch.where(ignored, torch.zeros_like(ez), 2 * ez + (512 + 8 * big) * U)
    if grad is None:
        return (lp,), (e,)
    half, tiny = HALF[hidden.dtype]
    p = torch.exp(z - lse[:, None])
    dz = -p
    dz[rows, ys] += 1
    g = torch.where(ignored, torch.zeros_like(lp), grad.double()) * scale
    dz = dz * g[:, None]
    # of a gradient's elements: both roundings, and the probability's own error
    edz = dz.abs() * (2 * half + 8 * U) + (p * (2 * ez + (512 + 8 * big) * U)[:, None]) * g.abs()[:, None]
    # fp16: relative to the largest row weight, half its least subnormal each time
    least = tiny * (2 * g.abs().nan_to_num().max() if hidden.dtype == torch.float16 else 1.0)
    edz = edz + 2 * least
    dz[bad] = math.nan
    gh, gw = dz @ w, dz.t() @ h
    # the products' own sums in fp32, and one rounding of the result
    egh = edz @ w.abs() + (dz.abs() @ w.abs()) * (2 * w.shape[0] * U) + half * gh.abs() + tiny
    egw = edz.t() @ h.abs() + (dz.abs().t() @ h.abs()) * (half + 2 * len(labels) * U) + half * gw.abs() + tiny
    if hidden.dtype == torch.float16:   # of the weighted hidden rows; no element of D is over 1
        egw = egw + len(labels) * least
    return (lp, gh, gw), (e, egh * 1.01, egw * 1.01)


def near(got, want, bound):
    """Every element within its bound, or NaN with a NaN wanted."""
    got = got.double()
    ok = ((got - want).abs() <= bound) | (got.isnan() & torch.as_tensor(want).isnan()) | (got == want)
    assert ok.all(), f"{int((~ok).sum())} of {ok.numel()} off, by up to {((got - want).abs() / bound)[~ok].max()} bounds"
