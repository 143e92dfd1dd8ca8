"""Activation checkpoints in 8 bits: half the bytes over the host link and in
pinned host memory.

The reference's checkpoints cross the link in the model's type
(sliding_checkpoint.py:69-73, 105); this format is an addition.  Blocks of 128
consecutive elements share a scale ``a / T``, ``a`` the largest magnitude of
the block and ``T`` the largest code: 127 of ``"int8"``, 448 of ``"fp8"``
(e4m3).  ``int8`` errs by at most ``a / 254``, ``fp8`` by a sixteenth of the
element itself, which is the better one where a block holds a few outliers.  A
block with an infinity or a NaN comes back as NaNs.

On a host, and for what the kernels cannot read through a pointer (a traced
call, a batch of a vmap), the same steps run as torch operations.  The packing
is not differentiable: a checkpoint's gradient is that of what it restores.
"""

from __future__ import annotations

import contextlib
import math
from typing import Optional, Sequence

import torch

from . import _native
from .fused_ce import _PLAIN, _memory_is_value, _traced
from .kernels import _CE_DTYPES, _stream_ptr

BLOCK = _native.SF_ACT8_BLOCK
FORMATS = {"int8": _native.SF_ACT8_INT8, "fp8": _native.SF_ACT8_FP8}
_TOP = {"int8": 127.0, "fp8": 448.0}
_LEAST, _MOST = 2.0 ** -100, float.fromhex("0x1.fffff0p127")


def act8_bytes(numel: int) -> int:
    """Bytes of ``numel`` packed elements."""
    return -(-numel // BLOCK) * _native.SF_ACT8_BLOCK_BYTES


def _check_format(fmt: str) -> int:
    if fmt not in FORMATS:
        raise ValueError(f"8-bit checkpoint format must be one of {sorted(FORMATS)}, got {fmt!r}")
    return FORMATS[fmt]


def _reads_memory(t: torch.Tensor) -> bool:
    return t.is_cuda and not _traced() and type(t) in _PLAIN and _memory_is_value(t)


def _aligned(packed: torch.Tensor) -> bool:
    return packed.data_ptr() % 16 == 0


def _on(stream: Optional[torch.cuda.Stream]):
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def pack_act8(x: torch.Tensor, fmt: str = "int8", out: Optional[torch.Tensor] = None,
              stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """The elements of ``x`` (float32, bfloat16 or float16; in order, whatever
    its strides) packed into ``out``: uint8, ``act8_bytes(x.numel())`` of them,
    contiguous, made here if not given (one that starts on no 16-byte boundary
    takes a copy more).  Asynchronous on ``stream`` (default: the current one)."""
    code = _check_format(fmt)
    if x.dtype not in _CE_DTYPES:
        raise TypeError(f"pack_act8: float32, bfloat16 or float16 expected, got {x.dtype}")
    n = x.numel()
    nbytes = act8_bytes(n)
    if out is not None and (out.dtype != torch.uint8 or out.numel() != nbytes or not out.is_contiguous()
                            or out.device != x.device):
        raise ValueError(f"pack_act8: out must be {nbytes} contiguous uint8 on {x.device}")
    if out is None and stream is None and n > 0 and x.is_cuda and not _traced():
        packed = _native.ops().act8_pack(x, _CE_DTYPES[x.dtype], code, nbytes)
        if packed is not None:
            return packed
    x = x.detach()
    if not _reads_memory(x) or (out is not None and not _reads_memory(out)):
        packed = _pack_torch(x, fmt)
        return packed if out is None else out.copy_(packed.view(out.shape))
    if x.device.index != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return pack_act8(x, fmt, out, stream)
    with _on(stream):   # what is made here belongs to that stream
        packed = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if out is None or not _aligned(out) else out
        x = x.contiguous()
        if n:
            _native.check(_native.hip().sf_act8_pack(x.data_ptr(), _CE_DTYPES[x.dtype], n, packed.data_ptr(), code,
                                                     _stream_ptr(stream)), "sf_act8_pack")
        return packed if out is None or packed is out else out.copy_(packed.view(out.shape))


def unpack_act8(packed: torch.Tensor, shape: Sequence[int], dtype: torch.dtype = torch.bfloat16, fmt: str = "int8",
                out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """What ``pack_act8`` packed, as a tensor of ``shape`` and ``dtype``, into
    the contiguous ``out`` if given.  A ``packed`` that starts on no 16-byte
    boundary takes a copy more."""
    code = _check_format(fmt)
    if dtype not in _CE_DTYPES:
        raise TypeError(f"unpack_act8: float32, bfloat16 or float16 expected, got {dtype}")
    shape = torch.Size(shape)
    if out is None and stream is None and packed.is_cuda and not _traced():
        x = _native.ops().act8_unpack(packed, shape, _CE_DTYPES[dtype], code)
        if x is not None:
            return x
    n = math.prod(shape)
    if packed.dtype != torch.uint8 or packed.numel() != act8_bytes(n) or not packed.is_contiguous():
        raise ValueError(f"unpack_act8: {act8_bytes(n)} contiguous uint8 expected for {tuple(shape)}")
    if out is not None and (out.dtype != dtype or out.shape != shape or not out.is_contiguous()
                            or out.device != packed.device):
        raise ValueError(f"unpack_act8: out must be a contiguous {dtype} tensor of {tuple(shape)} on {packed.device}")
    if not _reads_memory(packed) or (out is not None and not _reads_memory(out)):
        x = _unpack_torch(packed, n, dtype, fmt).view(shape)
        return x if out is None else out.copy_(x)
    if packed.device.index != torch.cuda.current_device():
        with torch.cuda.device(packed.device):
            return unpack_act8(packed, shape, dtype, fmt, out, stream)
    with _on(stream):
        out = torch.empty(shape, dtype=dtype, device=packed.device) if out is None else out
        packed = packed if _aligned(packed) else packed.clone()
        if n:
            _native.check(_native.hip().sf_act8_unpack(packed.data_ptr(), code, n, out.data_ptr(), _CE_DTYPES[dtype],
                                                       _stream_ptr(stream)), "sf_act8_unpack")
    return out


def _pack_torch(x: torch.Tensor, fmt: str) -> torch.Tensor:
    flat = x.reshape(-1).float()
    blocks = torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)
    most = blocks.abs().amax(dim=1, keepdim=True)
    finite = torch.isfinite(most)
    most = most.clamp(_LEAST, _MOST)
    top = torch.full_like(most, _TOP[fmt])
    scaled = torch.where(finite, blocks * torch.div(top, most), torch.zeros_like(blocks))
    scale = torch.where(finite, torch.div(most, top), torch.full_like(most, math.nan))
    codes = scaled.round().to(torch.int8) if fmt == "int8" else scaled.to(torch.float8_e4m3fn)
    return torch.cat([codes.view(torch.uint8).reshape(-1), scale.reshape(-1).view(torch.uint8)])


def _unpack_torch(packed: torch.Tensor, n: int, dtype: torch.dtype, fmt: str) -> torch.Tensor:
    nblocks = -(-n // BLOCK)
    packed = packed.reshape(-1)
    codes = packed[:nblocks * BLOCK].view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()
    scale = packed[nblocks * BLOCK:].clone().view(torch.float32)
    return (codes.view(nblocks, BLOCK) * scale.unsqueeze(1)).view(-1)[:n].to(dtype)
