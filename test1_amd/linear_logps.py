"""Log-probabilities of given tokens under the output unit, without keeping
its [N, V] logits: ``log_softmax(hidden @ weight.T / temperature)`` at the
labels, in fp32, with the gradients of the hidden rows and of the weight.

The reference's output unit gives the cross entropy or all logits
(slide_fsdp.py:77-113); losses over sequences of tokens need the
log-probabilities themselves, of the policy with gradients and of a reference
or an old policy without.

Numerics: the logits stay fp32 (they are not rounded to 16 bits in between),
maximum and sum of the softmax are fp32, and the gradient of the logits is
rounded to the inputs' type once, for its two products.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .alignment import _on_device, _stream
from .fused_ce import _DTYPES, _PLAIN, _memory_is_value, _traced
from .kernels import _CE_DTYPES


def _f32_out(dtype: torch.dtype) -> dict:
    return {} if dtype == torch.float32 else dict(out_dtype=torch.float32)


def _chunk_rows(vocab: int) -> int:
    """Rows whose fp32 logits take 1 GiB."""
    return max(1, (1 << 28) // vocab)


def _logits_buffer(rows: int, vocab: int, device) -> torch.Tensor:
    return torch.empty((rows, -(-vocab // 64) * 64), dtype=torch.float32, device=device)


def _forward_kernels(hidden, weight, labels, ignore_index, scale):
    n, v = hidden.shape[0], weight.shape[0]
    step = min(n, _chunk_rows(v))
    buf = _logits_buffer(step, v, hidden.device)
    lse = torch.empty(n, dtype=torch.float32, device=hidden.device)
    logp = torch.empty(n, dtype=torch.float32, device=hidden.device)
    wt = weight.t()
    for s in range(0, n, step):
        e = min(n, s + step)
        torch.mm(hidden[s:e], wt, **_f32_out(hidden.dtype), out=buf[:e - s, :v])
        _native.check(_native.hip().sf_logps_rows(
            buf.data_ptr(), buf.stride(0), e - s, v, labels.data_ptr() + 8 * s, ignore_index, scale,
            lse.data_ptr() + 4 * s, logp.data_ptr() + 4 * s, _stream()), "sf_logps_rows")
    return logp, lse


def _rescale(out: torch.Tensor, grad: torch.Tensor, norm: torch.Tensor) -> torch.Tensor:
    """``out`` = the fp32 ``grad`` over ``norm[0]``, rounded once."""
    _native.check(_native.hip().sf_ce_scale(norm.data_ptr() + 4, norm.data_ptr() + 8, None, None, 0, grad.data_ptr(),
                                            out.data_ptr(), out.numel(), _CE_DTYPES[out.dtype], _stream()),
                  "sf_ce_scale")
    return out


def _backward_kernels(grad, hidden, weight, labels, lse, ignore_index, scale, need_hidden, need_weight):
    n, h = hidden.shape
    v = weight.shape[0]
    dev, dtype = hidden.device, hidden.dtype
    f32 = _f32_out(dtype)
    step = min(n, _chunk_rows(v))
    buf = _logits_buffer(step, v, dev)
    dz_buf = buf if dtype == torch.float32 else torch.empty(buf.shape, dtype=dtype, device=dev)
    norm = None
    if dtype == torch.float16:
        norm = torch.empty(3, dtype=torch.float32, device=dev)
        _native.check(_native.hip().sf_logps_norm(grad.data_ptr(), labels.data_ptr(), ignore_index, n, scale,
                                                  norm.data_ptr(), _stream()), "sf_logps_norm")
    wide = norm is not None   # products into fp32, for the factor to leave before the rounding
    gh = torch.empty((n, h), dtype=torch.float32 if wide else dtype, device=dev) if need_hidden else None
    one = step == n and not wide
    gw = torch.empty((v, h), dtype=dtype if one else torch.float32, device=dev) if need_weight else None
    wt = weight.t()
    for s in range(0, n, step):
        e = min(n, s + step)
        torch.mm(hidden[s:e], wt, **f32, out=buf[:e - s, :v])
        dz = dz_buf[:e - s, :v]
        _native.check(_native.hip().sf_logps_grad(
            buf.data_ptr(), buf.stride(0), e - s, v, labels.data_ptr() + 8 * s, ignore_index, scale,
            lse.data_ptr() + 4 * s, grad.data_ptr() + 4 * s, norm.data_ptr() if wide else None, dz_buf.data_ptr(),
            _CE_DTYPES[dtype], dz_buf.stride(0), _stream()), "sf_logps_grad")
        if need_hidden:
            torch.mm(dz, weight, **(f32 if wide else {}), out=gh[s:e])
        if not need_weight:
            continue
        if one:
            torch.mm(dz.t(), hidden, out=gw)
        elif s == 0:
            torch.mm(dz.t(), hidden[s:e], **f32, out=gw)
        else:
            torch.addmm(gw, dz.t(), hidden[s:e], **f32, out=gw)
    if wide:
        gh = None if gh is None else _rescale(torch.empty((n, h), dtype=dtype, device=dev), gh, norm)
        gw = None if gw is None else _rescale(torch.empty((v, h), dtype=dtype, device=dev), gw, norm)
    return gh, None if gw is None else gw.to(dtype)


class _LinearLogps(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, scale):
        ctx.set_materialize_grads(False)
        logp, lse = _forward_kernels(hidden, weight, labels, ignore_index, scale)
        ctx.save_for_backward(hidden, weight, labels, lse)
        ctx.ignore_index, ctx.scale = ignore_index, scale
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return None, None, None, None, None
        hidden, weight, labels, lse = ctx.saved_tensors
        need = ctx.needs_input_grad[:2]
        if (type(grad) is torch.Tensor and _memory_is_value(grad) and _kernels_take(hidden, weight, labels)
                and lse.dtype == torch.float32 and lse.is_contiguous() and labels.is_contiguous()):
            with _on_device(hidden):
                return (*_backward_kernels(grad.to(torch.float32).contiguous(), hidden, weight, labels, lse,
                                           ctx.ignore_index, ctx.scale, *need), None, None, None)
        with torch.autocast(hidden.device.type, enabled=False):
            valid, at, bad = _label_kinds(labels, weight.shape[0], ctx.ignore_index)
            p = torch.exp(hidden.float() @ weight.float().t() * ctx.scale - lse.float().unsqueeze(1))
            onehot = torch.nn.functional.one_hot(at, weight.shape[0]).to(p.dtype)
            dz = (onehot - p) * (grad.to(torch.float32) * ctx.scale).unsqueeze(-1)
            dz = torch.where(valid.unsqueeze(1), dz, torch.zeros_like(dz))
            dz = torch.where(bad.unsqueeze(1), torch.full_like(dz, math.nan), dz)
            gh = (dz @ weight.float()).to(hidden.dtype) if need[0] else None
            gw = (dz.transpose(-1, -2) @ hidden.float()).to(weight.dtype) if need[1] else None
        return gh, gw, None, None, None


def _label_kinds(labels, vocab, ignore_index):
    valid = labels != ignore_index
    inside = (labels >= 0) & (labels < vocab)
    return valid, torch.where(valid & inside, labels, torch.zeros_like(labels)), valid & ~inside


def _torch_logps(hidden, weight, labels, ignore_index, scale):
    with torch.autocast(hidden.device.type, enabled=False):
        valid, at, bad = _label_kinds(labels, weight.shape[0], ignore_index)
        logp = torch.log_softmax(hidden.float() @ weight.float().t() * scale, dim=-1)
        logp = logp.gather(-1, at.unsqueeze(-1)).squeeze(-1)
        logp = logp * torch.where(bad, math.nan, 1.0)
        return torch.where(valid, logp, torch.zeros_like(logp))


def _kernels_take(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor) -> bool:
    return (hidden.is_cuda and not _traced() and hidden.numel() > 0 and weight.numel() > 0
            and weight.shape[0] <= 1 << 30 and labels.numel() < 1 << 31
            and weight.dtype == hidden.dtype and labels.dtype == torch.int64
            and weight.device == hidden.device and labels.device == hidden.device
            and all(type(t) in _PLAIN and _memory_is_value(t) for t in (hidden, weight, labels)))


def linear_logps(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100,
                 temperature: float = 1.0) -> torch.Tensor:
    """``log_softmax(hidden @ weight.T / temperature)`` at ``labels``, float32,
    of the labels' shape.

    ``hidden`` [..., H] and ``weight`` [V, H] of one float type (bfloat16,
    float16 or float32), ``labels`` [...] int64.  0, without gradient, where
    the label is ``ignore_index``; NaN where it is outside the vocabulary.
    Differentiable once by ``hidden`` and ``weight``; under ``no_grad`` nothing
    is kept.  Autocast does not change it."""
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError("linear_logps: hidden [..., H] and weight [V, H] expected")
    if labels.shape != hidden.shape[:-1]:
        raise ValueError("linear_logps: one label per hidden row expected")
    if hidden.dtype not in _DTYPES or weight.dtype != hidden.dtype:
        raise TypeError(f"linear_logps: hidden and weight of one float type expected, got {hidden.dtype}, {weight.dtype}")
    if labels.dtype != torch.int64:
        raise TypeError(f"linear_logps: int64 labels expected, got {labels.dtype}")
    if weight.device != hidden.device or labels.device != hidden.device:
        raise ValueError("linear_logps: hidden, weight and labels have to be on one device")
    if weight.shape[0] == 0:
        raise ValueError("linear_logps: an empty vocabulary")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError("linear_logps: temperature must be above 0")
    ignore_index, scale = int(ignore_index), 1.0 / float(temperature)
    if not _kernels_take(hidden, weight, labels):
        return _torch_logps(hidden, weight, labels, ignore_index, scale)
    rows = hidden.reshape(-1, hidden.shape[-1]) if hidden.dim() != 2 else hidden
    flat = labels.reshape(-1).contiguous()
    with _on_device(hidden):
        if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
            logp = _LinearLogps.apply(rows, weight, flat, ignore_index, scale)
        else:
            logp = _forward_kernels(rows, weight, flat, ignore_index, scale)[0]
    return logp if labels.dim() == 1 else logp.view(labels.shape)
