"""The largest log-probabilities of rows of logits, and one token drawn from each
row after temperature, top-k, top-p and min-p.

The reference trains on given tokens alone (slide_fsdp.py:85-113).  What a
teacher leaves for distillation is ``top_logps`` of its logits; the answers
that ``policy_loss`` takes, with their log-probabilities under the policy that
sampled them, come from ``sample_tokens``.

The kernels (``csrc/sf_sample.hip``) read the logits once, a sampled row's
border again, and sort no vocabulary.  What a draw is decided by is summed in 64
bits, as in exact arithmetic; the mass of all words, which log-probabilities
take, too, but of calls whose words are listed (``top_logps``, draws of the
largest or of up to 128): there each lane sums up to 64 words in fp32.
Logits that are large over the temperature, masks of any finite value among
them, cost no accuracy.  On a host, and for calls that the
kernels cannot serve (traced, batched by vmap), the same runs as torch
operations.  Neither is differentiable.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Union

import torch

from . import _native
from .fused_ce import _DTYPES, _traced

TOP_MOST = _native.SF_TOP_MOST     # words that top_logps gives at most


class TopLogps(NamedTuple):
    logps: torch.Tensor    # [..., k] float32, falling
    ids: torch.Tensor      # [..., k] int64


class SampledTokens(NamedTuple):
    ids: torch.Tensor      # [...] int64
    logps: torch.Tensor    # [...] float32


def _check_logits(what: str, logits: torch.Tensor) -> None:
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"{what}: logits of [..., vocabulary] expected, got {tuple(logits.shape)}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"{what}: bfloat16, float16 or float32 logits expected, got {logits.dtype}")


def _lse(z: torch.Tensor) -> torch.Tensor:
    return torch.logsumexp(z, dim=-1, keepdim=True)


def _bad(logits: torch.Tensor) -> torch.Tensor:
    """Rows without a distribution: a NaN, +infinity, nothing but -infinity."""
    top = logits.amax(dim=-1)
    return top.isnan() | top.isinf()


def _top_torch(logits, k, temperature):
    bad = _bad(logits).unsqueeze(-1)
    order = torch.where(bad, torch.zeros_like(logits), logits).sort(dim=-1, descending=True, stable=True).indices[..., :k]
    z = torch.where(bad, 0.0, logits.double())
    z = (z - z.amax(dim=-1, keepdim=True)) / temperature   # or a low temperature's lse loses the sum
    logps = (z.gather(-1, order) - _lse(z)).float()
    return TopLogps(torch.where(bad, math.nan, logps), torch.where(bad, -1, order))


def top_logps(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogps:
    """The ``k`` largest of ``log_softmax(logits / temperature)`` along the last
    dimension and their words, by falling logit, the first of equals first.

    ``logits`` [..., V] bfloat16, float16 or float32; ``k`` from 1 to
    ``TOP_MOST`` (128) and V; ``temperature`` above 0 (beyond 1e-30 and 1e30 as
    those).  A row with a NaN or
    +infinity, or of -infinities alone, gives NaN and -1.  No gradient."""
    _check_logits("top_logps", logits)
    k = int(k)
    if not 1 <= k <= min(TOP_MOST, logits.shape[-1]):
        raise ValueError(f"top_logps: k from 1 to {min(TOP_MOST, logits.shape[-1])} expected, got {k}")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError("top_logps: temperature must be above 0")
    logits = logits.detach()
    if logits.is_cuda and logits.numel() > 0 and not _traced():
        out = _native.ops().top_logps(logits, k, float(temperature))
        if out is not None:
            return TopLogps(*out)
    return _top_torch(logits, k, min(max(float(temperature), 1e-30), 1e30))   # as the kernels take it


# ---------------------------------------------------------------------------
def _sample_torch(logits, uniforms, temperature, top_k, top_p, min_p):
    def each(x):   # a setting of each row, or of all
        return x.unsqueeze(-1) if isinstance(x, torch.Tensor) else torch.full_like(uniforms, x, dtype=torch.float64).unsqueeze(-1)

    bad = _bad(logits).unsqueeze(-1)
    x = torch.where(bad, torch.zeros_like(logits), logits)
    temperature, top_k, top_p, min_p = each(temperature).double(), each(top_k), each(top_p).double(), each(min_p).double()
    greedy = ~(temperature > 0)
    temperature = torch.where(greedy, 1.0, temperature.clamp(1e-30, 1e30))
    top_k = torch.where(greedy, 1, top_k)
    s, order = x.sort(dim=-1, descending=True, stable=True)
    s = s.double()
    w = ((s - s[..., :1]) / temperature).exp()
    at = torch.arange(x.shape[-1], device=x.device)
    first = at == 0
    kept = (top_k <= 0) | (at < top_k)
    mass = torch.where(kept, w, 0.0)
    before = mass.cumsum(dim=-1) - mass
    kept = kept & (~(top_p < 1) | (before < top_p * mass.sum(dim=-1, keepdim=True)) | first)
    kept = kept & (~(min_p > 0) | (w >= min_p) | (w == 1))
    mass = torch.zeros_like(w).scatter(-1, order, torch.where(kept, w, 0.0))
    upto = mass.cumsum(dim=-1)
    u = uniforms.double().unsqueeze(-1)
    u = torch.where(u > 0, u.clamp(max=1.0 - 2.0 ** -24), 0.0)
    over = (upto > u * upto[..., -1:]) & (mass > 0)
    last = torch.where(mass > 0, at, -1).amax(dim=-1, keepdim=True)
    ids = torch.where(over.any(dim=-1, keepdim=True), over.to(torch.int8).argmax(dim=-1, keepdim=True), last)
    logps = ((x.gather(-1, ids).double() - s[..., :1]) / temperature - w.sum(dim=-1, keepdim=True).log()).float()
    return SampledTokens(torch.where(bad, -1, ids).squeeze(-1), torch.where(bad, math.nan, logps).squeeze(-1))


def _setting(name: str, x, shape, device, dtype, least: float, most: float):
    """(value for all rows, value of each row or None)."""
    if isinstance(x, torch.Tensor) and x.dim() > 0:
        if x.shape != shape or x.device != device:
            raise ValueError(f"sample_tokens: {name} of every row has to be {tuple(shape)} on {device}")
        if x.dtype != dtype:
            raise TypeError(f"sample_tokens: {dtype} {name} of every row expected, got {x.dtype}")
        return 0, x.detach()
    value = int(x) if dtype == torch.int64 else float(x)
    if not (least <= value <= most and math.isfinite(value)) or value != x:
        raise ValueError(f"sample_tokens: {name} from {least} to {most} expected, got {x}")
    return value, None


def _check_draw(shape, device, uniforms: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The settings of a draw for ``shape`` rows, each (value for all, value of each row or None)."""
    if uniforms.shape != shape or uniforms.device != device:
        raise ValueError(f"sample_tokens: uniforms have to be {tuple(shape)} on {device}")
    if uniforms.dtype != torch.float32:
        raise TypeError(f"sample_tokens: float32 uniforms expected, got {uniforms.dtype}")
    return (_setting("temperature", temperature, shape, device, torch.float32, 0.0, 3.0e38),
            _setting("top_k", top_k, shape, device, torch.int64, 0, 2 ** 62),
            _setting("top_p", top_p, shape, device, torch.float32, 0.0, 1.0),
            _setting("min_p", min_p, shape, device, torch.float32, 0.0, 1.0))


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
                  min_p: Union[float, torch.Tensor] = 0.0) -> SampledTokens:
    """One token for each row of ``logits`` [..., V], drawn by ``uniforms`` [...]
    (float32, in [0, 1)), with its log-probability under ``softmax(logits /
    temperature)`` of all words.

    Words are ordered by falling logit, the first of equals first; with w =
    exp((logit - largest) / temperature) a row keeps the first ``top_k`` (0:
    all), of those the words with less than ``top_p`` of their mass before them
    (at least the first), and of those the words with w >= ``min_p``.  Drawn
    is the first kept word, by its index, with whom the sum of w exceeds
    ``uniforms`` times the kept mass: the same numbers draw the same tokens.

    Each setting is a number, or a tensor [...] of every row's own (float32,
    ``top_k`` int64).  ``temperature`` 0 takes the first of the largest words,
    its log-probability being that at temperature 1.  Rows' own settings are
    not checked: a temperature that is not above 0 counts as 0, a ``top_k``
    below 1 as none, a ``top_p`` from 1 and a ``min_p`` to 0 as none; a uniform
    outside [0, 1) as the nearest within.

    A row with a NaN or +infinity, or of -infinities alone, gives -1 and NaN.
    No gradient."""
    _check_logits("sample_tokens", logits)
    (t, ts), (k, ks), (p, ps), (m, ms) = _check_draw(logits.shape[:-1], logits.device, uniforms, temperature, top_k, top_p,
                                                     min_p)
    logits, uniforms = logits.detach(), uniforms.detach()
    if logits.is_cuda and logits.numel() > 0 and not _traced():
        out = _native.ops().sample_tokens(logits, uniforms, t, ts, k, ks, p, ps, m, ms)
        if out is not None:
            return SampledTokens(*out)
    return _sample_torch(logits, uniforms, *(v if own is None else own for v, own in ((t, ts), (k, ks), (p, ps), (m, ms))))
