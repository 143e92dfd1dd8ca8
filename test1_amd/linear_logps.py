"""Log-probabilities of given tokens under the output unit, without keeping
its [N, V] logits: ``log_softmax(hidden @ weight.T / temperature)`` at the
labels, in fp32, with the gradients of the hidden rows and of the weight.

The reference's output unit gives the cross entropy or all logits
(slide_fsdp.py:77-113); losses over sequences of tokens need the
log-probabilities themselves, of the policy with gradients and of a reference
or an old policy without.

Numerics: the logits stay fp32 (they are not rounded to 16 bits in between),
maximum and sum of the softmax are fp32.  The gradient's products take 16-bit
operands, fp32 of fp32 ones: the exponentials, kept to 16 bits relative to their
span of the vocabulary, and their share of 1 - p, rounded again (fp16 with a
factor of 2^14, which keeps them out of its subnormals); the label's
element is exact, and the rows' own factors stay fp32 up to the hidden rows of
the weight gradient's product.
"""

from __future__ import annotations

import contextlib
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .fused_ce import _DTYPES, _PLAIN, _memory_is_value, _saved_plain, _tiles, _traced
from .kernels import _CE_DTYPES


_SPAN = _native.SF_LOGPS_SPAN
# What the forward keeps for the backward at most, 2 bytes a logit, and what a
# backward that makes it again takes at a time.  Keeping it saves one of four
# products: forward and backward kept | again, ms, bf16, 4092 tokens x 4096 x
# 128256 10.3 | 13.4, 8190 x 5120 x 152064 30.2 | 44.6 (in chunks, whose weight
# gradients are summed in fp32: 2.3 GB kept, 5.0 GB for the chunk and the sum),
# 16380 x 2048 x 128256 21.6 | 29.7.  8 GiB is a thirty-sixth of the device's
# memory and holds 30,000 tokens of a vocabulary of 128256; what a backward in
# chunks takes does not grow with the tokens.
_KEEP_BYTES = 8 << 30
_AGAIN_BYTES = 2 << 30
# Tiles of 64 x 64 hidden elements that the launch transposing them takes.
_TURNED_TILES = 1 << 23


def _backward_rows(n: int, vocab: int, hidden: int) -> Tuple[int, bool]:
    """Rows that the backward takes at a time, and whether the forward keeps
    their exponentials for it (then all)."""
    row = 2 * (-(-vocab // _SPAN) * _SPAN)
    most = _TURNED_TILES // -(-hidden // 64) * 64
    step = min(max(64, _AGAIN_BYTES // row // 64 * 64), most)
    return (n, True) if (n + 63) * row <= _KEEP_BYTES and n <= most else (min(n, step), False)


def _hidden_parts(rows: int, weight: torch.Tensor) -> int:
    """Parts in which the hidden gradient's product sums over the vocabulary.
    The library sums each of its tiles in one workgroup, so up to 64 tiles of
    256 x 256 as many parts as give every compute unit one, at most 16 and of
    2000 words or more; us, one product | parts, tokens x hidden x vocabulary: 3
    x 512 x 59040 107 | 20 (16), 32 x 768 x 50257 120 | 40 (16), 16 x 4096 x
    128256 421 | 173 (16), 200 x 1024 x 32000 103 | 30 (16), 400 x 1024 x 16000
    70 | 29 (8), 834 x 896 x 6640 45 | 30 (2), 1000 x 2048 x 32000 279 | 122 (8),
    500 x 4096 x 128256 849 | 458 (8), 2000 x 2048 x 32000 388 | 212 (4).  Beyond,
    where the product is the framework's own, by how well the tiles fill rounds
    of 256 compute units, with what adding the parts up costs (1250 parts / V of
    the product); us, 2 | 4 | 8 | 16 parts: 8190 x 5120 x 152064 (640 tiles) 9616 |
    9762 | - | -, in one 10931, 8190 x 2560 x 50257 (320) 1797 | 1674 | 1772 | -,
    2046 x 2560 x 151936 (80) - | 1749 | 1408 | 1310, 6000 x 1024 x 32000 (96) 394 |
    411 | 333 | -, 4000 x 3584 x 152064 (224) - | 3725 | 3484 | 3593.  Whole rounds
    need none: 4092 x 4096 x 128256 3081, in two 3155."""
    v, h = weight.shape
    tiles = _tiles(rows, h)
    if (v < 4000 or weight.element_size() != 2 or h % 8 != 0 or not weight.is_contiguous()
            or weight.data_ptr() % 16 != 0 or rows * h >= 1 << 31):
        return 1
    able = [p for p in (1, 2, 4, 8, 16) if p == 1 or v >= 2000 * p]
    if tiles <= 64:
        return max(p for p in able if p == 1 or tiles * p <= 256)
    return min(able, key=lambda p: -(-tiles * p // 256) * 256 / (tiles * p) + (1250 * p / v if p > 1 else 0))


def _f32_out(dtype: torch.dtype) -> dict:
    return {} if dtype == torch.float32 else dict(out_dtype=torch.float32)


def _stream() -> int:
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _on_device(t: torch.Tensor):
    """The tensors' device as the current one, without cost where it is."""
    return _HERE if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


_HERE = contextlib.nullcontext()


def _chunk_rows(vocab: int) -> int:
    """Rows whose fp32 logits take 1 GiB."""
    return max(1, (1 << 28) // vocab)


def _logits_buffer(rows: int, vocab: int, device) -> torch.Tensor:
    return torch.empty((rows, -(-vocab // 64) * 64), dtype=torch.float32, device=device)


def _forward_kernels(hidden, weight, labels, ignore_index, scale):
    n, v = hidden.shape[0], weight.shape[0]
    lse = torch.empty(n, dtype=torch.float32, device=hidden.device)
    logp = torch.empty(n, dtype=torch.float32, device=hidden.device)
    step = min(n, _chunk_rows(v))
    buf = _logits_buffer(step, v, hidden.device)
    wt = weight.t()
    for s in range(0, n, step):
        e = min(n, s + step)
        torch.mm(hidden[s:e], wt, **_f32_out(hidden.dtype), out=buf[:e - s, :v])
        _native.check(_native.hip().sf_logps_rows(
            buf.data_ptr(), buf.stride(0), e - s, v, labels.data_ptr() + 8 * s, ignore_index, scale,
            lse.data_ptr() + 4 * s, logp.data_ptr() + 4 * s, _stream()), "sf_logps_rows")
    return logp, lse


def _row_weight(grad, logp, labels, vocab, ignore_index, scale, dtype):
    """What multiplies the rows of D, and what takes out fp16's factors (``sf_logps_weight``)."""
    n = labels.shape[0]
    weight = torch.empty(n, dtype=torch.float32, device=grad.device)
    norm = torch.empty(2, dtype=torch.float32, device=grad.device) if dtype == torch.float16 else None
    _native.check(_native.hip().sf_logps_weight(grad.data_ptr(), logp.data_ptr(), labels.data_ptr(), ignore_index, n,
                                                vocab, scale, weight.data_ptr(),
                                                None if norm is None else norm.data_ptr(), _stream()),
                  "sf_logps_weight")
    return weight, norm


def _add_product(total, a, b, first):
    """``total`` (+)= a @ b in fp32 or, of the only one, in the operands' type."""
    f32 = _f32_out(a.dtype) if total.dtype == torch.float32 else {}
    if first:
        torch.mm(a, b, **f32, out=total)
    else:
        torch.addmm(total, a, b, **f32, out=total)


def _rescaled(grad: Optional[torch.Tensor], dtype, norm) -> Optional[torch.Tensor]:
    """The weight gradient in ``dtype``, fp16's factor taken out before the rounding."""
    if grad is None or grad.dtype == dtype and norm is None:
        return grad
    if norm is None:
        return grad.to(dtype)
    out = torch.empty(grad.shape, dtype=dtype, device=grad.device)
    _native.check(_native.hip().sf_ce_scale(norm.data_ptr(), norm.data_ptr() + 4, None, None, 0, grad.data_ptr(),
                                            out.data_ptr(), out.numel(), _CE_DTYPES[dtype], _stream()), "sf_ce_scale")
    return out


def _backward_kernels(grad, hidden, weight, labels, logp, lse, ignore_index, scale, need_hidden, need_weight):
    n, h = hidden.shape
    v = weight.shape[0]
    dev, dtype = hidden.device, hidden.dtype
    row_weight, norm = _row_weight(grad, logp, labels, v, ignore_index, scale, dtype)
    row_weight = row_weight.unsqueeze(1)
    step = min(n, _chunk_rows(v))
    one = step == n
    buf = _logits_buffer(step, v, dev)
    d_buf = buf if dtype == torch.float32 else torch.empty(buf.shape, dtype=dtype, device=dev)
    gh = torch.empty((n, h), dtype=torch.float32, device=dev) if need_hidden else None
    gw = None
    if need_weight:
        gw = torch.empty((v, h), dtype=dtype if one and norm is None else torch.float32, device=dev)
        weighted = (hidden.masked_fill(row_weight == 0, 0) * row_weight).to(dtype)
    wt = weight.t()
    for s in range(0, n, step):
        e = min(n, s + step)
        torch.mm(hidden[s:e], wt, **_f32_out(dtype), out=buf[:e - s, :v])
        d = d_buf[:e - s, :v]
        _native.check(_native.hip().sf_logps_grad(
            buf.data_ptr(), buf.stride(0), e - s, v, labels.data_ptr() + 8 * s, ignore_index, scale,
            lse.data_ptr() + 4 * s, logp.data_ptr() + 4 * s, grad.data_ptr() + 4 * s, d_buf.data_ptr(),
            _CE_DTYPES[dtype], d_buf.stride(0), _stream()), "sf_logps_grad")
        if need_hidden:
            torch.mm(d, weight, **_f32_out(dtype), out=gh[s:e])
        if need_weight:
            _add_product(gw, d.t(), weighted[s:e], s == 0)
    if need_hidden:
        gh.masked_fill_(row_weight == 0, 0).mul_(row_weight)
        gh = (gh if norm is None else gh.mul_(norm[0])).to(dtype)
    return gh, _rescaled(gw, dtype, norm)


class _LinearLogps(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, scale):
        ctx.set_materialize_grads(False)
        logp, lse = _forward_kernels(hidden, weight, labels, ignore_index, scale)
        ctx.save_for_backward(hidden, weight, labels, lse, logp)
        ctx.ignore_index, ctx.scale = ignore_index, scale
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return None, None, None, None, None
        hidden, weight, labels, lse, logp = ctx.saved_tensors
        need = ctx.needs_input_grad[:2]
        if (type(grad) is torch.Tensor and grad.is_cuda and _memory_is_value(grad) and _kernels_take(hidden, weight, labels)
                and _saved_plain(lse, torch.float32, hidden.device) and _saved_plain(logp, torch.float32, hidden.device)
                and labels.is_contiguous()):
            with _on_device(hidden):
                return (*_backward_kernels(grad.to(torch.float32).contiguous(), hidden, weight, labels, logp, lse,
                                           ctx.ignore_index, ctx.scale, *need), None, None, None)
        with torch.autocast(hidden.device.type, enabled=False):
            valid, at, bad = _label_kinds(labels, weight.shape[0], ctx.ignore_index)
            counts = (valid & (grad != 0)).unsqueeze(-1)
            hidden32 = torch.where(counts, hidden.float(), torch.zeros((), device=hidden.device))
            p = torch.exp(hidden32 @ weight.float().t() * ctx.scale - lse.float().unsqueeze(1))
            onehot = torch.nn.functional.one_hot(at, weight.shape[0]).to(p.dtype)
            dz = (onehot - p) * (grad.to(torch.float32) * ctx.scale).unsqueeze(-1)
            dz = torch.where(counts, dz, torch.zeros_like(dz))
            dz = torch.where(counts & bad.unsqueeze(-1), torch.full_like(dz, math.nan), dz)
            gh = (dz @ weight.float()).to(hidden.dtype) if need[0] else None
            gw = (dz.transpose(-1, -2) @ hidden32).to(weight.dtype) if need[1] else None
        return gh, gw, None, None, None


def _label_kinds(labels, vocab, ignore_index):
    valid = labels != ignore_index
    inside = (labels >= 0) & (labels < vocab)
    return valid, torch.where(valid & inside, labels, torch.zeros_like(labels)), valid & ~inside


def _torch_logps(hidden, weight, labels, ignore_index, scale, bias=None):
    with torch.autocast(hidden.device.type, enabled=False):
        valid, at, bad = _label_kinds(labels, weight.shape[0], ignore_index)
        # what ignored tokens hold does not reach the weight's gradient
        hidden = torch.where(valid.unsqueeze(-1), hidden, torch.zeros_like(hidden))
        logits = hidden.float() @ weight.float().t()
        if bias is not None:
            logits = logits + bias.float()
        logp = torch.log_softmax(logits * scale, dim=-1)
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
    of the labels' shape.  On a GPU, tokens that are ignored or whose upstream
    gradient is 0 leave the gradients alone, whatever their hidden states hold.

    ``hidden`` [..., H] and ``weight`` [V, H] of one float type (bfloat16,
    float16 or float32), ``labels`` [...] int64.  0, without gradient, where
    the label is ``ignore_index``; NaN where it is outside the vocabulary.
    Differentiable once by ``hidden`` and ``weight``; under ``no_grad`` nothing
    is kept.  Autocast does not change it.  Logits over the temperature are
    fp32: the results are off by 2^-24 of their magnitude, and NaN where that is 2^31
    or more (a temperature of 1e-9 or so)."""
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
    need_grad = torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)
    step, keep, nparts = rows.shape[0], False, 1
    if need_grad:
        step, keep = _backward_rows(step, *weight.shape)
        nparts = _hidden_parts(step, weight)
    logp = _native.ops().linear_logps(rows, weight, flat, ignore_index, scale, nparts, step, keep)
    if logp is None:
        with _on_device(hidden):
            if need_grad:
                logp = _LinearLogps.apply(rows, weight, flat, ignore_index, scale)
            else:
                logp = _forward_kernels(rows, weight, flat, ignore_index, scale)[0]
    return logp if labels.dim() == 1 else logp.view(labels.shape)
