"""Cross entropy and log probabilities of a linear head, and their gradients.

``linear_cross_entropy``      loss and log-sum-exp of each token of x . W^T
``linear_cross_entropy_bwd``  dX and dW for given gradients of the losses
``linear_log_probs``          log probability of each given token, the entropy of its
                              distribution and the most likely alternatives
``linear_log_probs_bwd``      dX and dW for gradients of the first two

They take the place of the reference's two passes over vocabulary tiles
(doublepass/src/loss.rs, doublepass/kernels/fused_ce.cu:71-207): the logits live
in the accumulators of a tile, the gradients are computed in pieces of the
vocabulary.  The cross entropy never stores the logits; ``linear_log_probs`` keeps
them in fp32 for its gradients, by default while they take no more memory than W
(``keep_logits``: a pass that only scores says False).  x is bf16 [M, d] (the final
norm's output), W the bf16 head [V, d], targets int64 [M]; losses and log-sum-exp
are fp32.  The gradient of the logits is an operand of bf16 products and is rounded
to bf16 (2^-8 of each entry at most), as a bf16 model's own backward pass would; the
sums over it are fp32.
"""
from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .gemm import _workspace_for
from .nf4 import _ptr, _require_cuda, _run, _stream_ptr

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


def _check_dw(dw: Optional[torch.Tensor], accumulate: bool, w: torch.Tensor,
              x: torch.Tensor) -> torch.Tensor:
    """The gradient of w: what the caller gave, if it can be that, or new memory."""
    if dw is None:
        if accumulate:
            raise ValueError("accumulate needs an existing float32 dw")
        dw = torch.empty_like(w)
    if dw.dtype not in (torch.bfloat16, torch.float32) or dw.shape != w.shape \
            or dw.device != x.device:
        raise ValueError(f"dw must be bfloat16 or float32 {list(w.shape)} on x's device")
    if accumulate and dw.dtype != torch.float32:
        raise ValueError("accumulate needs a float32 dw")
    return dw


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
    dw = _check_dw(dw, accumulate, w, x)
    dx = torch.empty_like(x)
    workspace = _workspace_for(_workspace_bytes(m, v, d, True, x.get_device()), workspace, x)
    _lib.check(_lib.load().nf4s_linear_ce_bwd(
        x.data_ptr(), w.data_ptr(), targets.data_ptr(), lse.data_ptr(), dloss.data_ptr(), m, v, d,
        ignore_index, dx.data_ptr(), dw.data_ptr(), int(dw.dtype == torch.float32),
        int(accumulate), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
        _stream_ptr(x)))
    return dx, dw


TOP = 32  # alternatives of a token at most


@dataclass
class LogProbs:
    """Outputs of :func:`linear_log_probs`."""

    logp: torch.Tensor                # float32 [M], of the given tokens
    entropy: torch.Tensor             # float32 [M]
    lse: torch.Tensor                 # float32 [M]
    top_logp: Optional[torch.Tensor]  # float32 [M, top_k], with top_k > 0
    top_ids: Optional[torch.Tensor]   # int64 [M, top_k]
    logits: Optional[torch.Tensor] = None  # float32, in the kernels' order, if kept
    shape: Optional[Tuple[int, int, int]] = None  # tokens, V and d of kept logits


def log_probs_workspace_bytes(m: int, v: int, d: int, top_k: int = 0,
                              backward: bool = False) -> int:
    """Workspace of :func:`linear_log_probs`, or of its gradients, for M tokens and a
    [V, d] head."""
    return _log_probs_workspace_bytes(m, v, d, top_k, backward, torch.cuda.current_device())


@functools.lru_cache(maxsize=256)
def _log_probs_workspace_bytes(m: int, v: int, d: int, top_k: int, backward: bool,
                               device: int) -> int:
    out = ctypes.c_int64(0)
    _run(device, _lib.load().nf4s_linear_logprob_workspace_size, m, v, d, top_k, int(backward),
         ctypes.byref(out))
    return int(out.value)


@functools.lru_cache(maxsize=256)
def _logits_bytes(m: int, v: int, d: int, device: int) -> int:
    out = ctypes.c_int64(0)
    _run(device, _lib.load().nf4s_linear_logprob_logits_size, m, v, d, ctypes.byref(out))
    return int(out.value)


def linear_log_probs(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, top_k: int = 0,
                     ignore_index: int = IGNORE_INDEX,
                     workspace: Optional[torch.Tensor] = None,
                     keep_logits: Optional[bool] = None) -> LogProbs:
    """Log probability of ``targets`` under softmax(x . W^T), the entropy and the
    log-sum-exp of every token, and with ``top_k`` (up to 32) the tokens of largest
    logit in order, equal ones by their index, with their log probabilities.  A target
    equal to ``ignore_index`` (no token is given) has logp 0, and the rest as any
    other; a target outside [0, V) has NaN (it is only seen on the device).  A row with
    a NaN logit, or an infinite largest one, is NaN in everything but ``top_ids`` (and
    the log-sum-exp of -inf alone, -inf).

    ``keep_logits``: the result holds the logits in fp32, and the gradients need not
    multiply x . W^T again (a quarter of a training pass' products).  By default
    (None) where no alternatives are asked for and they take no more memory than W,
    which is up to d / 2 tokens, 16384 at most; they live as long as the result.  A pass
    that only scores saves 4 M V bytes (2.1 GB at 4096 tokens, 128000 columns) and up to
    a seventh of its time with False."""
    _check_head(x, w, targets)
    m, d, v = int(x.shape[0]), int(x.shape[1]), int(w.shape[0])
    top_k = int(top_k)
    if not 0 <= top_k <= min(TOP, v):
        raise ValueError(f"top_k must be 0 to {TOP} and at most {v}, got {top_k}")
    logp = torch.empty(m, dtype=torch.float32, device=x.device)
    lse, entropy = torch.empty_like(logp), torch.empty_like(logp)
    top_logp = top_ids = None
    if top_k > 0:
        top_logp = torch.empty(m, top_k, dtype=torch.float32, device=x.device)
        top_ids = torch.empty(m, top_k, dtype=torch.int64, device=x.device)
    logits = None
    if keep_logits or (keep_logits is None and top_k == 0 and 2 * m <= d):
        need = _logits_bytes(m, v, d, x.get_device())
        if keep_logits and m > 0 and (top_k > 0 or need == 0):
            raise ValueError("logits are kept without alternatives, of up to 16384 tokens")
        if need > 0:
            logits = torch.empty(need // 4, dtype=torch.float32, device=x.device)
    workspace = _workspace_for(
        _log_probs_workspace_bytes(m, v, d, top_k, False, x.get_device()), workspace, x)
    _run(x.get_device(), _lib.load().nf4s_linear_logprob_fwd, x.data_ptr(), w.data_ptr(),
         targets.data_ptr(), m, v, d, top_k, ignore_index, logp.data_ptr(), lse.data_ptr(),
         entropy.data_ptr(), _ptr(top_logp), _ptr(top_ids), _ptr(logits), workspace.data_ptr(),
         workspace.numel() * workspace.element_size(), _stream_ptr(x))
    return LogProbs(logp, entropy, lse, top_logp, top_ids, logits,
                    None if logits is None else (m, v, d))


def linear_log_probs_bwd(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, out: LogProbs,
                         dlogp: torch.Tensor, dentropy: Optional[torch.Tensor] = None,
                         ignore_index: int = IGNORE_INDEX, dw: Optional[torch.Tensor] = None,
                         accumulate: bool = False, workspace: Optional[torch.Tensor] = None
                         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dx bf16 [M, d], dw [V, d]) for the gradients ``dlogp`` and ``dentropy`` (fp32
    [M]; None: zero) of :func:`linear_log_probs`' result ``out``.  An ignored target's
    dlogp does not count, its dentropy does.  dw is bf16 unless a float32 ``dw`` is
    given, which the micro-batches of a step may ``accumulate`` into; the gradients of
    the logits enter both products rounded to bf16, as in
    :func:`linear_cross_entropy_bwd`, divided by the largest ``|dlogp|``.  Kept logits
    are the forward's: of x and W as they were then, and of these sizes (``out.shape``).
    Tokens with both gradients zero count as zeros times their row of x, which has to be
    finite."""
    _check_head(x, w, targets)
    _require_cuda(out.lse, out.entropy, dlogp, dentropy, dw)
    m, d, v = int(x.shape[0]), int(x.shape[1]), int(w.shape[0])
    for t, name in ((out.lse, "lse"), (out.entropy, "entropy"), (dlogp, "dlogp"),
                    (dentropy, "dentropy")):
        if t is not None and (t.dtype != torch.float32 or list(t.shape) != [m]
                              or t.device != x.device):
            raise ValueError(f"{name} must be float32 [{m}] on x's device")
    logits = out.logits
    if logits is not None:
        _require_cuda(logits)
        # Their order goes by all three sizes, other ones may have as many.
        if logits.dtype != torch.float32 or logits.device != x.device or out.shape != (m, v, d) \
                or logits.numel() * 4 != _logits_bytes(m, v, d, x.get_device()):
            raise ValueError("out's logits are of another head, or of other tokens")
    dw = _check_dw(dw, accumulate, w, x)
    dx = torch.empty_like(x)
    workspace = _workspace_for(
        _log_probs_workspace_bytes(m, v, d, 0, True, x.get_device()), workspace, x)
    _run(x.get_device(), _lib.load().nf4s_linear_logprob_bwd, x.data_ptr(), w.data_ptr(),
         targets.data_ptr(), out.lse.data_ptr(), out.entropy.data_ptr(), _ptr(logits),
         dlogp.data_ptr(), _ptr(dentropy), m, v, d, ignore_index, dx.data_ptr(), dw.data_ptr(),
         int(dw.dtype == torch.float32), int(accumulate), workspace.data_ptr(),
         workspace.numel() * workspace.element_size(), _stream_ptr(x))
    return dx, dw
