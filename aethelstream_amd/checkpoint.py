"""Activation checkpoints in 8 bits, and the recompute that starts from one.

The first pass of a double-pass step keeps each layer's input for the second;
the reference compresses it to int8 per channel (doublepass/src/checkpoint.rs
:21-60, ramflow/kernels/checkpoint_compress.cu:53-145).  Here 128 elements along
a row share an fp32 scale: 1.03 bytes an element.

``encode``       activation (fp32 or bf16) -> :class:`Checkpoint8`
``decode``       back to fp32 or bf16
``decode_norm``  decode and RMSNorm in one pass: the recompute's first step
                 (doublepass/src/backward.rs:438-447), residual and GEMM operand
``norm.block_norm_bwd`` reads a :class:`Checkpoint8` in the residual's place.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .nf4 import _ptr, _require_cuda, _stream_ptr

EPS = 1e-6   # of the norm (math.rs:45)
BLOCK = 128  # elements of a row that share a scale


@dataclass
class Checkpoint8:
    """A checkpointed activation [M, d]: values are codes * their block's scale."""

    codes: torch.Tensor   # int8 [M, d]
    scales: torch.Tensor  # float32 [M, ceil(d / 128)]

    def check(self) -> None:
        """Raises unless codes and scales belong together on one device."""
        c, s = self.codes, self.scales
        if not (c.is_contiguous() and s.is_contiguous() and c.is_cuda):
            _require_cuda(c, s)
        if c.dtype is not torch.int8 or s.dtype is not torch.float32:
            raise ValueError("checkpoint codes must be int8 and scales float32")
        if c.dim() != 2 or c.device != s.device:
            raise ValueError("checkpoint codes must be [M, d], with scales on their device")
        m, d = c.shape
        if s.shape != (m, (d + BLOCK - 1) // BLOCK):
            raise ValueError(f"checkpoint scales must be [{m}, {(d + BLOCK - 1) // BLOCK}], got "
                             f"{list(s.shape)}")


def encode(x: torch.Tensor, out: Optional[Checkpoint8] = None) -> Checkpoint8:
    """Checkpoint of x [M, d], fp32 or bf16, into ``out`` if given.  A block of
    128 that holds an infinity or a NaN reads back as NaN."""
    _require_cuda(x)
    if x.dtype not in (torch.float32, torch.bfloat16) or x.dim() != 2:
        raise ValueError("x must be a float32 or bfloat16 [M, d] tensor")
    m, d = int(x.shape[0]), int(x.shape[1])
    if out is None:
        out = Checkpoint8(torch.empty_like(x, dtype=torch.int8),
                          torch.empty(m, (d + BLOCK - 1) // BLOCK, dtype=torch.float32,
                                      device=x.device))
    else:
        out.check()
        if out.codes.device != x.device or out.codes.shape != x.shape:
            raise ValueError("out must hold x's shape on x's device")
    _lib.check(_lib.load().nf4s_ckpt8_encode(x.data_ptr(), int(x.dtype == torch.bfloat16), m, d,
                                             out.codes.data_ptr(), out.scales.data_ptr(),
                                             _stream_ptr(x)))
    return out


def decode(ckpt: Checkpoint8, dtype: torch.dtype = torch.float32,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The checkpointed values in ``dtype`` (float32 or bfloat16), or in ``out``'s."""
    ckpt.check()
    if out is None:
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("checkpoints decode to float32 or bfloat16")
        out = torch.empty_like(ckpt.codes, dtype=dtype)
    _require_cuda(out)
    if out.dtype not in (torch.float32, torch.bfloat16) or out.shape != ckpt.codes.shape \
            or out.device != ckpt.codes.device:
        raise ValueError("out must be a float32 or bfloat16 tensor of the checkpoint's shape and "
                         "device")
    m, d = ckpt.codes.shape
    _lib.check(_lib.load().nf4s_ckpt8_decode(ckpt.codes.data_ptr(), ckpt.scales.data_ptr(), m, d,
                                             out.data_ptr(), int(out.dtype == torch.bfloat16),
                                             _stream_ptr(out)))
    return out


def decode_norm(ckpt: Checkpoint8, w: torch.Tensor, eps: float = EPS, want_x: bool = True
                ) -> Tuple[Optional[torch.Tensor], torch.Tensor, torch.Tensor]:
    """(x fp32 [M, d] or None, y bf16 [M, d], rms fp32 [M]): the checkpointed
    residual and its RMSNorm, from one read of the codes."""
    ckpt.check()
    _require_cuda(w)
    m, d = ckpt.codes.shape
    dev = ckpt.codes.device
    if w.dtype != torch.float32 or list(w.shape) != [d] or w.device != dev:
        raise ValueError(f"w must be float32 [{d}] on the checkpoint's device")
    x = torch.empty_like(ckpt.codes, dtype=torch.float32) if want_x else None
    y = torch.empty_like(ckpt.codes, dtype=torch.bfloat16)
    rms = torch.empty(m, dtype=torch.float32, device=dev)
    _lib.check(_lib.load().nf4s_ckpt8_decode_norm(ckpt.codes.data_ptr(), ckpt.scales.data_ptr(),
                                                  w.data_ptr(), m, d, float(eps), _ptr(x),
                                                  y.data_ptr(), rms.data_ptr(), _stream_ptr(y)))
    return x, y, rms
