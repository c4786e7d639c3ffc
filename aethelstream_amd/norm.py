"""RMSNorm forward on the device, producing the fused GEMMs' bf16 operand.

``rms_norm_fwd`` replaces rms_norm_fwd (doublepass/src/math.rs:28-59) at
single_layer_forward's two call sites (doublepass/src/forward.rs:173, 249),
whose output is the input of the q/k/v and gate/up GEMMs.  The reference
returns (y, x_hat, rms) in fp32; here y leaves as bf16 (the GEMM operand) and
rms as fp32 (x_hat = x / rms is recomputed where the backward needs it).

``block_norm_fwd`` / ``block_norm_bwd`` are the whole boundary between two
blocks: an optional norm of the block's output, a gate per channel and a
residual scale, the residual add and the next block's norm (forward.rs:249).
Without a block ``block_norm_bwd`` is the backward of rms_norm_fwd.
"""
from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .checkpoint import Checkpoint8
from .gemm import _workspace_for
from .nf4 import _ptr, _require_cuda, _stream_ptr

EPS = 1e-6  # math.rs:45


def rms_norm_fwd(x: torch.Tensor, w: torch.Tensor, eps: float = EPS,
                 out: Optional[torch.Tensor] = None,
                 rms: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [M, d] fp32, w [d] fp32 -> (y [M, d] bf16, rms [M] fp32)."""
    _require_cuda(x, w)
    if x.dtype != torch.float32 or w.dtype != torch.float32:
        raise ValueError("x and w must be float32")
    if x.dim() != 2 or w.dim() != 1 or w.shape[0] != x.shape[1]:
        raise ValueError(f"x must be [M, d] and w [d], got {list(x.shape)} and {list(w.shape)}")
    if not x.is_contiguous() or not w.is_contiguous():
        raise ValueError("x and w must be contiguous")
    m, d = int(x.shape[0]), int(x.shape[1])
    if out is None:
        out = torch.empty(m, d, dtype=torch.bfloat16, device=x.device)
    if rms is None:
        rms = torch.empty(m, dtype=torch.float32, device=x.device)
    # A caller's out / rms is written by the kernel: it must be contiguous
    # device memory on x's device (a host tensor's pointer would reach the
    # kernel, a strided one would be overwritten as if contiguous).
    _require_cuda(out, rms)
    if out.device != x.device or rms.device != x.device:
        raise ValueError("out and rms must be on x's device")
    if out.dtype != torch.bfloat16 or list(out.shape) != [m, d]:
        raise ValueError("out must be a contiguous bfloat16 [M, d] tensor")
    if rms.dtype != torch.float32 or rms.numel() < m:
        raise ValueError("rms must hold M float32 values")
    _lib.check(_lib.load().nf4s_rmsnorm_fwd(x.data_ptr(), w.data_ptr(), m, d, float(eps),
                                            out.data_ptr(), rms.data_ptr(), _stream_ptr(x)))
    return out, rms


@dataclass
class BlockNorm:
    """Outputs of :func:`block_norm_fwd`."""

    res: torch.Tensor                 # float32 [M, d], the new residual
    y: torch.Tensor                   # bfloat16 [M, d], its norm: the next block's input
    rms_pre: torch.Tensor             # float32 [M], of res
    rms_post: Optional[torch.Tensor]  # float32 [M], of h (with w_post)


@dataclass
class BlockNormGrad:
    """Outputs of :func:`block_norm_bwd`."""

    dres: torch.Tensor                # float32 [M, d], of the residual that came in
    dh: Optional[torch.Tensor]        # bfloat16 [M, d], of the block's output
    dw_pre: torch.Tensor              # float32 [d]
    dw_post: Optional[torch.Tensor]   # float32 [d]
    dgate: Optional[torch.Tensor]     # float32 [d]


def _check_rows(t: Optional[torch.Tensor], name: str, dtype: torch.dtype, shape: tuple,
                device: torch.device) -> None:
    """Raises unless t is None or a contiguous tensor of that type, shape and device."""
    if t is None or (t.dtype is dtype and t.shape == shape and t.device == device
                     and t.is_contiguous()):
        return
    _require_cuda(t)
    raise ValueError(f"{name} must be {str(dtype)[6:]} {list(shape)} on {device}, got "
                     f"{str(t.dtype)[6:]} {list(t.shape)} on {t.device}")


@functools.lru_cache(maxsize=256)
def _bwd_workspace_bytes(m: int, d: int, device: int) -> int:
    size = ctypes.c_int64()
    _lib.check(_lib.load().nf4s_block_norm_bwd_workspace_size(m, d, ctypes.byref(size)))
    return size.value


def block_norm_fwd(h: torch.Tensor, res: torch.Tensor, w_pre: torch.Tensor,
                   w_post: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                   alpha: float = 1.0, eps: float = EPS,
                   out: Optional[torch.Tensor] = None) -> BlockNorm:
    """The boundary after a block with output h (bf16 [M, d]) and residual res
    (fp32 [M, d]):

        u = w_post * h / rms(h)  (u = h without w_post)
        res' = res + alpha * gate * u  (gate 1 without one)
        y = w_pre * res' / rms(res')

    in one pass.  w_pre, w_post and gate are fp32 [d].  The new residual goes to
    ``out`` if given, which may be ``res``."""
    _require_cuda(h)
    if h.dim() != 2:
        raise ValueError(f"h must be [M, d], got {list(h.shape)}")
    m, d = rows = h.shape
    dev = h.device
    _check_rows(h, "h", torch.bfloat16, rows, dev)
    _check_rows(res, "res", torch.float32, rows, dev)
    for t, name in ((w_pre, "w_pre"), (w_post, "w_post"), (gate, "gate")):
        _check_rows(t, name, torch.float32, (d,), dev)
    if out is None:
        out = torch.empty_like(res)
    else:
        _check_rows(out, "out", torch.float32, rows, dev)
    y = torch.empty_like(h)
    rms_pre = torch.empty(m, dtype=torch.float32, device=dev)
    rms_post = None if w_post is None else torch.empty_like(rms_pre)
    _lib.check(_lib.load().nf4s_block_norm_fwd(
        h.data_ptr(), res.data_ptr(), w_pre.data_ptr(), _ptr(w_post), _ptr(gate), float(alpha), m,
        d, float(eps), out.data_ptr(), y.data_ptr(), rms_pre.data_ptr(), _ptr(rms_post),
        _stream_ptr(h)))
    return BlockNorm(out, y, rms_pre, rms_post)


def block_norm_bwd(dy: torch.Tensor, dres: Optional[torch.Tensor], res, rms_pre: torch.Tensor,
                   w_pre: torch.Tensor, h: Optional[torch.Tensor] = None,
                   rms_post: Optional[torch.Tensor] = None,
                   w_post: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                   alpha: float = 1.0, out: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None) -> BlockNormGrad:
    """Gradients of :func:`block_norm_fwd` for the gradients dy (bf16) of y and
    dres (fp32, None: zero) of the new residual.  ``res`` is the forward's new
    residual, fp32 or a :class:`aethelstream_amd.checkpoint.Checkpoint8` of it,
    rms_pre the rms of what ``res`` stands for.  Without ``h`` there is no block:
    the RMSNorm backward of res.  The residual's gradient goes to ``out`` if
    given, which may be ``dres``."""
    _require_cuda(dy)
    if dy.dim() != 2:
        raise ValueError(f"dy must be [M, d], got {list(dy.shape)}")
    m, d = rows = dy.shape
    dev = dy.device
    _check_rows(dy, "dy", torch.bfloat16, rows, dev)
    _check_rows(dres, "dres", torch.float32, rows, dev)
    codes = scales = None
    if isinstance(res, Checkpoint8):
        res.check()
        codes, scales, res = res.codes, res.scales, None
        if codes.shape != rows or codes.device != dev:
            raise ValueError(f"the checkpoint must be [{m}, {d}] on dy's device")
    elif res is None:
        raise ValueError("res must be a float32 tensor or a Checkpoint8")
    _check_rows(res, "res", torch.float32, rows, dev)
    _check_rows(rms_pre, "rms_pre", torch.float32, (m,), dev)
    for t, name in ((w_pre, "w_pre"), (w_post, "w_post"), (gate, "gate")):
        _check_rows(t, name, torch.float32, (d,), dev)
    if h is None and (w_post is not None or gate is not None):
        raise ValueError("w_post and gate need h")
    if w_post is not None and rms_post is None:
        raise ValueError("w_post needs rms_post")
    _check_rows(h, "h", torch.bfloat16, rows, dev)
    _check_rows(rms_post, "rms_post", torch.float32, (m,), dev)
    if out is None:
        out = torch.empty(m, d, dtype=torch.float32, device=dev)
    else:
        _check_rows(out, "out", torch.float32, rows, dev)
    dh = None if h is None else torch.empty_like(h)
    dw_pre = torch.empty_like(w_pre)
    dw_post = None if w_post is None else torch.empty_like(w_post)
    dgate = None if gate is None else torch.empty_like(gate)
    workspace = _workspace_for(_bwd_workspace_bytes(m, d, dev.index), workspace, dy)
    _lib.check(_lib.load().nf4s_block_norm_bwd(
        dy.data_ptr(), _ptr(dres), _ptr(res), _ptr(codes), _ptr(scales), rms_pre.data_ptr(),
        w_pre.data_ptr(), _ptr(h), _ptr(rms_post), _ptr(w_post), _ptr(gate), float(alpha), m, d,
        out.data_ptr(), _ptr(dh), dw_pre.data_ptr(), _ptr(dw_post), _ptr(dgate),
        workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream_ptr(dy)))
    return BlockNormGrad(out, dh, dw_pre, dw_post, dgate)
