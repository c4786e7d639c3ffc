"""An AdamW step over many tensors at once, with moments in 32 or in 8 bits.

``adamw_step``    one step of every tensor, in one launch for each mix of types
``adamw_state``   zero moments for given parameters
``moments``       what the moments are, in fp32
``coefficients``  a step's eight scalars, on the device for a captured step

The place of the reference's optimizer behind the weight gradients
(galore/kernels/quantize_state.cu:7-98, with one int8 scale a tensor).  Parameters
are fp32 or bf16; fp32 ones may leave bf16 copies in the same pass.  After a step a
layer's fp32 masters go to ``nf4.requantize_``.
"""
from __future__ import annotations

import ctypes
import operator
from array import array
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .nf4 import _ptr, _require_cuda, _run, _stream_ptr

BLOCK = 128  # elements that share a scale, and what every tensor's moments begin at
MOST_BETA_8 = 0.95  # beta1 and beta2 with 8-bit moments
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


@dataclass
class AdamWState:
    """Moments of tensors of the given sizes, one after the other in flat buffers,
    each from a multiple of 128 on (what lies between is zero): fp32, or 8-bit codes
    with one scale for 128 elements (``m`` int8, ``v`` uint8).

    In 8 bits m is off by at most 2^-4 of |m| + 2^-15 s, s its block's largest, and
    sqrt(v) by 2^-5 of sqrt(v) + 2^-15 s (2^-22 s beside for fp32's own roundings); one
    that is not zero is 2^-19 s at least, which may be up to that much too large.  A NaN
    or an infinity in a block's moments makes its scale, and so all 128 of them, NaN.

    Rounding is to nearest, so a change by less than half the distance of two codes is
    lost.  Steps therefore take beta1 and beta2 up to 0.95 (:data:`MOST_BETA_8`) with
    8-bit moments: there gradients that vary from step to step carry m and sqrt(v)
    along, within 1 % of 32 bits' on average, also after their size changed.  At beta2 =
    0.999 sqrt(v) of gradients that grew four times stays at half of what it should be,
    of a tenth at four times it; at beta1 = 0.98 m keeps the sign of a mean that turned.
    Gradients that hardly vary in size are followed badly at 0.95 too (they grew: sqrt(v)
    stays at 0.74; they fell to a tenth: it hardly falls): those need 32 bits.  With a
    gradient of zero |m| falls by a code's distance at least, so that a value whose
    gradients end comes to rest also where others of its block go on.  (Gradients of less
    than some 2^-16 of their block's largest, but not zero, are lost in m's codes.)"""

    sizes: List[int]
    m: torch.Tensor
    v: torch.Tensor
    m_scale: Optional[torch.Tensor] = None  # float32, one for 128 elements
    v_scale: Optional[torch.Tensor] = None  # ... of sqrt(v)

    @property
    def bits(self) -> int:
        return 32 if self.m_scale is None else 8

    def starts(self) -> List[int]:
        """Where each tensor's moments begin."""
        at, out = 0, []
        for n in self.sizes:
            out.append(at)
            at += (n + BLOCK - 1) // BLOCK * BLOCK
        return out

    def check(self) -> int:
        """Raises unless the buffers belong together; the blocks they hold."""
        blocks = sum((n + BLOCK - 1) // BLOCK for n in self.sizes)
        m, v = self.m, self.v
        _require_cuda(m, v, self.m_scale, self.v_scale)
        if (self.m_scale is None) != (self.v_scale is None):
            raise ValueError("m_scale and v_scale: both or neither")
        kinds = (torch.float32, torch.float32) if self.m_scale is None else (torch.int8,
                                                                             torch.uint8)
        if (m.dtype, v.dtype) != kinds or m.shape != (blocks * BLOCK,) or m.shape != v.shape \
                or m.device != v.device:
            raise ValueError(f"moments must be {kinds[0]} and {kinds[1]} [{blocks * BLOCK}] on one "
                             "device")
        for s in (self.m_scale, self.v_scale):
            if s is not None and (s.dtype != torch.float32 or s.shape != (blocks,)
                                  or s.device != m.device):
                raise ValueError(f"scales must be float32 [{blocks}] on the moments' device")
        return blocks


def adamw_state(params: Sequence[torch.Tensor], bits: int = 32) -> AdamWState:
    """Zero moments for ``params``, in 32 or 8 bits."""
    if bits not in (32, 8):
        raise ValueError("moments have 32 or 8 bits")
    if not params:
        raise ValueError("no parameters")
    dev = params[0].device
    sizes = [int(p.numel()) for p in params]
    blocks = sum((n + BLOCK - 1) // BLOCK for n in sizes)
    kinds = (torch.float32,) * 2 if bits == 32 else (torch.int8, torch.uint8)
    m, v = (torch.zeros(blocks * BLOCK, dtype=t, device=dev) for t in kinds)
    if bits == 32:
        return AdamWState(sizes, m, v)
    return AdamWState(sizes, m, v, torch.zeros(blocks, device=dev), torch.zeros(blocks, device=dev))


def coefficients(step: int, lr: float, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.0) -> List[float]:
    """The eight scalars of step ``step`` (from 1 on), computed in 64 bits: beta1,
    1 - beta1, beta2, 1 - beta2, 1 - lr wd, lr / (1 - beta1^t), 1 / sqrt(1 -
    beta2^t), eps.  A float32 device tensor of them is what a captured step takes as
    ``hyper``; the program writes each step's into it before the replay."""
    b1, b2 = betas
    if step < 1:
        raise ValueError("steps count from 1")
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
        raise ValueError("betas must lie in [0, 1)")
    if not (lr >= 0.0 and eps >= 0.0 and weight_decay >= 0.0):
        raise ValueError("lr, eps and weight_decay must not be negative")
    return [b1, 1.0 - b1, b2, 1.0 - b2, 1.0 - lr * weight_decay, lr / (1.0 - b1 ** step),
            (1.0 - b2 ** step) ** -0.5, eps]


_dtype = operator.attrgetter("dtype")
_numel, _same_size, _device = torch.Tensor.numel, torch.Tensor.is_same_size, torch.Tensor.get_device
_contiguous, _data_ptr = torch.Tensor.is_contiguous, torch.Tensor.data_ptr


def _refuse(p: torch.Tensor, g: torch.Tensor, c: Optional[torch.Tensor], n: int,
            dev: torch.device) -> None:
    """Raises if a tensor does not belong with its gradient, copy and moments."""
    _require_cuda(p, g, c)
    if p.numel() != n or g.shape != p.shape:
        raise ValueError(f"a parameter {list(p.shape)} with a gradient {list(g.shape)} and moments "
                         f"of {n}")
    if p.dtype not in _TYPES or g.dtype not in _TYPES:
        raise ValueError("parameters and gradients must be float32 or bfloat16")
    if c is not None and (c.dtype != torch.bfloat16 or p.dtype != torch.float32
                          or c.shape != p.shape):
        raise ValueError("a copy is bfloat16, of a float32 parameter's shape")
    if any(t is not None and t.device != dev for t in (p, g, c)):
        raise ValueError(f"every tensor must be on the moments' device {dev}")


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], state: AdamWState,
               step: int, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 0.0,
               grad_scale: Optional[torch.Tensor] = None,
               copies: Optional[Sequence[Optional[torch.Tensor]]] = None,
               hyper: Optional[torch.Tensor] = None) -> None:
    """Step ``step`` (from 1 on) of every parameter, in place, with decoupled weight
    decay: fp32 or bf16 parameters and gradients in any mix, contiguous.

    ``grad_scale``: float32 [1] on the device that multiplies every gradient (a
    clipping factor).  ``copies``: for each parameter None, or the bfloat16 tensor
    that gets the updated fp32 parameter.  ``hyper``: float32 [8] on the device,
    :func:`coefficients` of the step, in place of step, lr, betas, eps and
    weight_decay; a captured step needs it to take another step at its replay.

    8-bit moments need beta1 and beta2 of at most 0.95, so others than the default; in
    ``hyper``, which is only seen on the device, larger ones leave parameters and moments
    NaN."""
    count = len(state.sizes)
    if len(params) != count or len(grads) != count or \
            (copies is not None and len(copies) != count):
        raise ValueError(f"the state is of {count} tensors, got {len(params)} parameters and "
                         f"{len(grads)} gradients" +
                         ("" if copies is None else f", {len(copies)} copies"))
    state.check()
    dev = state.m.device
    index = state.m.get_device()
    # Whole lists at a time: of 241 tensors 0.1 ms, of which each is looked at alone
    # (0.16) only to say what is wrong.
    kinds = [list(map(_dtype, params)), list(map(_dtype, grads))]
    found = [list(map(_TYPES.get, k)) for k in kinds]
    if None in found[0] or None in found[1] or list(map(_numel, params)) != state.sizes \
            or not all(map(_same_size, params, grads)) \
            or set(map(_device, params)) | set(map(_device, grads)) != {index} \
            or not all(map(_contiguous, params)) or not all(map(_contiguous, grads)):
        for p, g, n in zip(params, grads, state.sizes):
            _refuse(p, g, None, n, dev)
    if copies is not None:
        for p, g, c, n in zip(params, grads, copies, state.sizes):
            if c is not None and (p.dtype is not torch.float32 or c.dtype is not torch.bfloat16
                                  or c.shape != p.shape or c.get_device() != index
                                  or not c.is_contiguous()):
                _refuse(p, g, c, n, dev)
    types = [a + 2 * b for a, b in zip(*found)]
    for t, n, name in ((grad_scale, 1, "grad_scale"), (hyper, 8, "hyper")):
        if t is not None:
            _require_cuda(t)
            if t.dtype != torch.float32 or t.numel() != n or t.device != dev:
                raise ValueError(f"{name} must be float32 [{n}] on the moments' device")
    host = None
    if hyper is None:
        if state.bits == 8 and max(betas) > MOST_BETA_8:
            raise ValueError(f"8-bit moments take beta1 and beta2 up to {MOST_BETA_8}, got {betas}:"
                             " the codes would not follow the gradients")
        host = (ctypes.c_float * 8)(*coefficients(step, lr, betas, eps, weight_decay))
    lists = [array("Q", map(_data_ptr, params)), array("Q", map(_data_ptr, grads)),
             None if copies is None else array("Q", [0 if c is None else c.data_ptr()
                                                     for c in copies]),
             array("q", state.sizes), array("i", types)]
    at = [None if a is None else a.buffer_info()[0] for a in lists]
    _run(index, _lib.load().nf4s_adamw_step, *at, count, state.m.data_ptr(), state.v.data_ptr(),
         _ptr(state.m_scale), _ptr(state.v_scale), host, _ptr(hyper), _ptr(grad_scale),
         _stream_ptr(state.m))


def moments(state: AdamWState) -> Tuple[torch.Tensor, torch.Tensor]:
    """m and v in fp32, laid out as in the state: its own buffers in 32 bits, what the
    codes stand for in 8."""
    blocks = state.check()
    if state.m_scale is None:
        return state.m, state.v
    m = torch.empty(blocks * BLOCK, dtype=torch.float32, device=state.m.device)
    v = torch.empty_like(m)
    _run(m.get_device(), _lib.load().nf4s_adamw_moments, state.m.data_ptr(), state.v.data_ptr(),
         state.m_scale.data_ptr(), state.v_scale.data_ptr(), blocks, m.data_ptr(), v.data_ptr(),
         _stream_ptr(m))
    return m, v
