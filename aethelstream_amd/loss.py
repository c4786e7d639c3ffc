"""Cross entropy of a linear head without keeping the logits, and its gradients.

``linear_cross_entropy``      loss and log-sum-exp of each token of x . W^T
``linear_cross_entropy_bwd``  dX and dW for given gradients of the losses

They take the place of the reference's two passes over vocabulary tiles
(doublepass/src/loss.rs, doublepass/kernels/fused_ce.cu:71-207): the logits live
in the accumulators of a tile, the gradients are computed in pieces of the
vocabulary.  x is bf16 [M, d] (the final norm's output), W the bf16 head [V, d],
targets int64 [M]; losses and log-sum-exp are fp32.  The gradient of the logits
is an operand of bf16 products and is rounded to bf16 (2^-8 of each entry at
most), as a bf16 model's own backward pass would; the sums over it are fp32.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch

from . import _lib
from .gemm import _workspace_for
from .nf4 import _require_cuda, _stream_ptr

IGNORE_INDEX = -100


def workspace_bytes(m: int, v: int, d: int, backward: bool) -> int:
    """Workspace of the forward, or of the gradients, for M tokens and a [V, d] head."""
    return _workspace_bytes(m, v, d, backward, torch.cuda.current_device())


@functools.lru_cache(maxsize=256)
def _workspace_bytes(m: int, v: int, d: int, backward: bool, device: int) -> int:
    out = ctypes.c_int64(0)
    _lib.check(_lib.load().nf4s_linear_ce_workspace_size(m, v, d, int(backward),
                                                         ctypes.byref(out)))
    return int(out.value)


def _check_head(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor) -> None:
    _require_cuda(x, w, targets)
    if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16:
        raise ValueError("x and w must be bfloat16")
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"x [M, d] and w [V, d] must share d, got {list(x.shape)} and "
                         f"{list(w.shape)}")
    if targets.dtype != torch.int64 or list(targets.shape) != [x.shape[0]]:
        raise ValueError(f"targets must be int64 [{x.shape[0]}]")
    if w.device != x.device or targets.device != x.device:
        raise ValueError("x, w and targets must be on one device")


def linear_cross_entropy(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor,
                         ignore_index: int = IGNORE_INDEX,
                         workspace: Optional[torch.Tensor] = None
                         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss [M], lse [M]) in fp32.  A target equal to ``ignore_index`` has loss
    0; any other outside [0, V) has loss NaN (it is only seen on the device).
    ``workspace``: a buffer to use instead of one from torch's caching allocator,
    if it holds :func:`workspace_bytes`."""
    _check_head(x, w, targets)
    m, d, v = int(x.shape[0]), int(x.shape[1]), int(w.shape[0])
    loss = torch.empty(m, dtype=torch.float32, device=x.device)
    lse = torch.empty_like(loss)
    workspace = _workspace_for(_workspace_bytes(m, v, d, False, x.get_device()), workspace, x)
    _lib.check(_lib.load().nf4s_linear_ce_fwd(
        x.data_ptr(), w.data_ptr(), targets.data_ptr(), m, v, d, ignore_index, loss.data_ptr(),
        lse.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
        _stream_ptr(x)))
    return loss, lse


def linear_cross_entropy_bwd(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor,
                             lse: torch.Tensor, dloss: torch.Tensor,
                             ignore_index: int = IGNORE_INDEX, dw: Optional[torch.Tensor] = None,
                             accumulate: bool = False,
                             workspace: Optional[torch.Tensor] = None
                             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dx bf16 [M, d], dw [V, d]) for the gradient ``dloss`` fp32 [M] of each
    token's loss.  dw is bf16 unless a float32 ``dw`` is given, which the
    micro-batches of a step may ``accumulate`` into: its sums are fp32 and are not
    rounded again, but the bf16 logit gradients that enter them leave rows that
    are no token's target about 0.0016 (relative) from the exact gradient, the
    targets' 0.0001.  They are held divided by the largest ``|dloss|``: tokens that
    share one ``dloss`` keep it exactly, with a ``dloss`` of their own they carry
    its rounding (targets' rows 0.0013).  Ignored tokens count as zeros times their
    row of x, which has to be finite."""
    _check_head(x, w, targets)
    _require_cuda(lse, dloss, dw)
    m, d, v = int(x.shape[0]), int(x.shape[1]), int(w.shape[0])
    for t, name in ((lse, "lse"), (dloss, "dloss")):
        if t.dtype != torch.float32 or list(t.shape) != [m] or t.device != x.device:
            raise ValueError(f"{name} must be float32 [{m}] on x's device")
    if dw is None:
        if accumulate:
            raise ValueError("accumulate needs an existing float32 dw")
        dw = torch.empty_like(w)
    if dw.dtype not in (torch.bfloat16, torch.float32) or list(dw.shape) != [v, d] \
            or dw.device != x.device:
        raise ValueError(f"dw must be bfloat16 or float32 [{v}, {d}] on x's device")
    if accumulate and dw.dtype != torch.float32:
        raise ValueError("accumulate needs a float32 dw")
    dx = torch.empty_like(x)
    workspace = _workspace_for(_workspace_bytes(m, v, d, True, x.get_device()), workspace, x)
    _lib.check(_lib.load().nf4s_linear_ce_bwd(
        x.data_ptr(), w.data_ptr(), targets.data_ptr(), lse.data_ptr(), dloss.data_ptr(), m, v, d,
        ignore_index, dx.data_ptr(), dw.data_ptr(), int(dw.dtype == torch.float32),
        int(accumulate), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
        _stream_ptr(x)))
    return dx, dw
