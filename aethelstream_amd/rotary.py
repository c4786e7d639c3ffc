"""Queries and keys between their products and attention: a norm for each head
and the rotation by position in one pass, or the rotation alone.

``apply``      q, k -> normed and rotated q, k
``apply_bwd``  their gradients, and those of the norms' weights
``Rotary``     the angles: :func:`frequencies` and :func:`Rotary.from_frequencies`

q and k are what ``gemm.linear_fwd_grouped`` leaves for a layer's q and k
projections (doublepass/src/forward.rs:174-176), as [M, heads, d] views: bf16 or
fp32, tokens and heads at any distance, a head's elements adjacent, so parts of one
wider row are taken where they lie.  Sums, norms and angles are fp32 or better;
results are rounded once.
"""
from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .gemm import _workspace_for
from .nf4 import _ptr, _run, _stream_ptr

EPS = 1e-6  # of the norms, as the layers' (math.rs:45)
MAX_HEAD = 1024
MAX_HEADS = 4096


def frequencies(rot: int, base: float = 10000.0, factor: float = 1.0,
                trained: Optional[int] = None, fast: float = 32.0, slow: float = 1.0
                ) -> Tuple[List[float], float]:
    """Radians a position of the rot / 2 pairs, ``base ** (-2 i / rot)``, and the
    factor of the rotated values (1).

    ``factor`` > 1 stretches them for contexts that many times longer than trained.
    Without ``trained`` every frequency is divided by it.  With the trained length,
    pairs that turn ``fast`` times or more within it keep theirs, those that turn
    ``slow`` times or less are divided, with a ramp in the index between (from a whole
    index to a whole one, be it outside the head), and the values grow by
    ``0.1 ln(factor) + 1``."""
    if rot <= 0 or rot % 2 != 0:
        raise ValueError(f"rot must be positive and even, got {rot}")
    if not (base > 0 and factor >= 1):
        raise ValueError("base must be positive and factor at least 1")
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if factor == 1:
        return f, 1.0
    if trained is None:
        return [v / factor for v in f], 1.0
    if not (fast > slow > 0 and trained > 0 and base > 1):
        raise ValueError("needs fast > slow > 0, trained > 0 and base > 1")

    def index(turns: float) -> float:  # of the pair that turns so often within `trained`
        return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    # The ramp may begin before the first pair or end behind the last: cut off there, it
    # would divide a last pair that turns often, or keep a first one that hardly does.
    low, high = math.floor(index(fast)), math.ceil(index(slow))
    # (One apart at least, but for a fast and a slow that rounding makes equal.)
    wide = max(high - low, 1)
    ramp = [min(max((i - low) / wide, 0.0), 1.0) for i in range(rot // 2)]
    return ([v * (1 - r) + v / factor * r for v, r in zip(f, ramp)],
            0.1 * math.log(factor) + 1.0)


@dataclass
class Rotary:
    """Angles of a rotation: ``turns`` int64 [rot / 2] on the device, turns a
    position of each pair in units of 2^-64 (so that position * turns modulo 2^64 is
    an exact fraction of a turn); pairs (i, i + rot / 2), or (2 i, 2 i + 1) if
    ``interleaved``; ``scale`` multiplies the rotated values."""

    turns: torch.Tensor
    interleaved: bool = False
    scale: float = 1.0

    @staticmethod
    def from_frequencies(radians: Sequence[float], interleaved: bool = False, scale: float = 1.0,
                         device: Optional[torch.device] = None) -> "Rotary":
        """Of radians a position, in 64 bits, one for each pair."""
        units = []
        for v in radians:
            if not math.isfinite(v):
                raise ValueError("frequencies must be finite")
            t = int(math.fmod(v / (2 * math.pi), 1.0) * 2.0 ** 64) % (1 << 64)
            units.append(t - (1 << 64) if t >= 1 << 63 else t)
        return Rotary(torch.tensor(units, dtype=torch.int64, device=device or "cuda"), interleaved,
                      scale)


@dataclass
class RotaryGrad:
    """Outputs of :func:`apply_bwd`."""

    dq: torch.Tensor
    dk: Optional[torch.Tensor]
    dw_q: Optional[torch.Tensor]  # float32 [d], with norms
    dw_k: Optional[torch.Tensor]


def _heads(t: torch.Tensor, name: str, ref: torch.Tensor, shape=None) -> None:
    if t.dim() != 3 or t.dtype != ref.dtype or t.device != ref.device or not t.is_cuda:
        raise ValueError(f"{name} must be a [M, heads, d] device tensor of the others' type")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError(f"the elements of a head of {name} must be adjacent")


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """The bytes from t's first element to its last."""
    first = t.data_ptr()
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return first, first + (last + 1) * t.element_size()


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.stride() == b.stride() and a.shape == b.shape


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether a and b lie apart: one behind the other, or side by side in rows of
    one length."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return True
    row = a.stride(0) * a.element_size()
    if a.stride(0) != b.stride(0) or min(a.stride(1), b.stride(1)) < 0 or row <= 0:
        return False
    wide = [((t.shape[1] - 1) * t.stride(1) + t.shape[2]) * t.element_size() for t in (a, b)]
    off = (b0 - a0) % row
    return off >= wide[0] and off + wide[1] <= row


def _check_out(out: torch.Tensor, name: str, own: Sequence[torch.Tensor],
               others: Sequence[torch.Tensor]) -> None:
    """Raises unless every element of out has a place of its own, and out lies apart
    from each of ``own`` or is it, and apart from all of ``others``."""
    if out.numel() == 0:
        return
    (m, h, d), (st, sh, _) = out.shape, out.stride()
    tokens = (h == 1 or sh >= d) and (m == 1 or st >= (h - 1) * sh + d)
    heads = (m == 1 or st >= d) and (h == 1 or sh >= (m - 1) * st + d)
    if not (tokens or heads):
        raise ValueError(f"{name} has elements that share a place")
    if not all(_same(out, t) or _apart(out, t) for t in own) \
            or not all(_apart(out, t) for t in others):
        raise ValueError(f"{name} overlaps another tensor that it is not")


def _explain(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rope: Rotary,
              w_q: Optional[torch.Tensor], w_k: Optional[torch.Tensor]) -> Tuple[int, ...]:
    """The shape (M, hq, hk, d) of arguments that belong together; raises for others."""
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("q and k must be bfloat16 or float32")
    _heads(q, "q", q)
    m, hq, d = q.shape
    hk = 0
    if k is not None:
        _heads(k, "k", q)
        if k.shape[0] != m or k.shape[2] != d:
            raise ValueError(f"q {list(q.shape)} and k {list(k.shape)} must share tokens and d")
        hk = k.shape[1]
        if hk == 0:
            raise ValueError("k has no heads: pass None")
    if hq == 0 or d == 0 or d % 2 != 0 or d > MAX_HEAD or max(hq, hk) > MAX_HEADS:
        raise ValueError(f"heads must have an even size up to {MAX_HEAD}, at most {MAX_HEADS} of "
                         f"them, got {hq} and {hk} of {d}")
    if positions.dtype != torch.int64 or positions.shape != (m,) or positions.device != q.device \
            or not positions.is_contiguous():
        raise ValueError(f"positions must be contiguous int64 [{m}] on q's device")
    t = rope.turns
    if t.dtype != torch.int64 or t.dim() != 1 or t.device != q.device or not t.is_contiguous():
        raise ValueError("the rotation's turns must be contiguous int64 [rot / 2] on q's device")
    if not 1 <= t.shape[0] <= d // 2:
        raise ValueError(f"the rotation turns {2 * t.shape[0]} of {d} elements")
    if k is not None and (w_q is None) != (w_k is None):
        raise ValueError("w_q and w_k: both or neither")
    if k is None and w_k is not None:
        raise ValueError("w_k needs k")
    for w, name in ((w_q, "w_q"), (w_k, "w_k")):
        if w is not None and (w.dtype != torch.float32 or w.shape != (d,) or w.device != q.device
                              or not w.is_contiguous()):
            raise ValueError(f"{name} must be contiguous float32 [{d}] on q's device")
    return m, hq, hk, d


def _check(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rope: Rotary,
           w_q: Optional[torch.Tensor], w_k: Optional[torch.Tensor]) -> Tuple[int, ...]:
    """:func:`_explain` in one condition where all is well, as ever but once: 1 us of a
    call of 9, for a kernel of 4."""
    shape, dtype, dev, t = q.shape, q.dtype, q.get_device(), rope.turns
    if len(shape) == 3 and k is not None and len(k.shape) == 3:
        m, hq, d = shape
        mk, hk, dk = k.shape
        if mk == m and dk == d and 0 < hq <= MAX_HEADS and 0 < hk <= MAX_HEADS \
                and 0 < d <= MAX_HEAD and d % 2 == 0 and q.stride(2) == 1 and k.stride(2) == 1 \
                and dev >= 0 and dev == k.get_device() == positions.get_device() == t.get_device() \
                and k.dtype is dtype and (dtype is torch.bfloat16 or dtype is torch.float32) \
                and positions.dtype is torch.int64 and t.dtype is torch.int64 \
                and positions.shape == (m,) and len(t.shape) == 1 and 0 < 2 * t.shape[0] <= d \
                and positions.is_contiguous() and t.is_contiguous() \
                and (w_q is None and w_k is None or w_q is not None and w_k is not None
                     and w_q.dtype is w_k.dtype is torch.float32
                     and w_q.get_device() == w_k.get_device() == dev
                     and w_q.shape == w_k.shape == (d,)
                     and w_q.is_contiguous() and w_k.is_contiguous()):
            return m, hq, hk, d
    return _explain(q, k, positions, rope, w_q, w_k)


_EIGHT, _TWELVE = ctypes.c_int64 * 8, ctypes.c_int64 * 12


def _pair(t: Optional[torch.Tensor]) -> Tuple[int, ...]:
    """The distances of t's tokens and heads."""
    return (0, 0) if t is None else t.stride()[:2]


def _empty(m: int, heads: int, d: int, like: torch.Tensor) -> torch.Tensor:
    if like.is_contiguous():
        return torch.empty_like(like)
    return torch.empty(m, heads, d, dtype=like.dtype, device=like.device)


def apply(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rope: Rotary,
          w_q: Optional[torch.Tensor] = None, w_k: Optional[torch.Tensor] = None,
          eps: float = EPS, out_q: Optional[torch.Tensor] = None,
          out_k: Optional[torch.Tensor] = None
          ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(q', k') of q [M, hq, d] and k [M, hk, d] (None: q alone) at ``positions``
    int64 [M]: every head normed with w_q or w_k (fp32 [d], both or neither; rms =
    sqrt(mean + eps)), then its first 2 * len(rope.turns) elements rotated.  They go
    to ``out_q`` and ``out_k`` if given, which may be q and k themselves; the backward
    with norms needs q and k as they were."""
    m, hq, hk, d = _check(q, k, positions, rope, w_q, w_k)
    if out_q is None:
        out_q = _empty(m, hq, d, q)
    else:
        _heads(out_q, "out_q", q, q.shape)
        _check_out(out_q, "out_q", [q], [] if k is None else [k])
    if k is None:
        if out_k is not None:
            raise ValueError("out_k needs k")
    elif out_k is None:
        out_k = _empty(m, hk, d, k)
    else:
        _heads(out_k, "out_k", q, k.shape)
        _check_out(out_k, "out_k", [k], [q, out_q])
    _run(q.get_device(), _lib.load().nf4s_rotary_fwd, q.data_ptr(), _ptr(k),
         int(q.dtype == torch.bfloat16), m, hq, hk, d,
         _EIGHT(*q.stride()[:2], *_pair(k), *out_q.stride()[:2], *_pair(out_k)), _ptr(w_q),
         _ptr(w_k), float(eps), positions.data_ptr(), rope.turns.data_ptr(),
         2 * rope.turns.shape[0], int(rope.interleaved), float(rope.scale), out_q.data_ptr(),
         _ptr(out_k), _stream_ptr(q))
    return out_q, out_k


@functools.lru_cache(maxsize=256)
def _bwd_workspace_bytes(m: int, hq: int, hk: int, d: int, device: int) -> int:
    size = ctypes.c_int64()
    _run(device, _lib.load().nf4s_rotary_bwd_workspace_size, m, hq, hk, d, ctypes.byref(size))
    return size.value


def apply_bwd(dq: torch.Tensor, dk: Optional[torch.Tensor], positions: torch.Tensor, rope: Rotary,
              q: Optional[torch.Tensor] = None, k: Optional[torch.Tensor] = None,
              w_q: Optional[torch.Tensor] = None, w_k: Optional[torch.Tensor] = None,
              eps: float = EPS, out_q: Optional[torch.Tensor] = None,
              out_k: Optional[torch.Tensor] = None,
              workspace: Optional[torch.Tensor] = None) -> RotaryGrad:
    """Gradients of :func:`apply` for the gradients dq and dk of its results.  With
    norms q and k are its inputs, and the weights' gradients, sums over all tokens
    and heads, are returned too; without, q and k are not read and may be None.  The
    gradients go to ``out_q`` and ``out_k`` if given, which may be dq and dk, or q
    and k."""
    m, hq, hk, d = _check(dq, dk, positions, rope, w_q, w_k)
    norm = w_q is not None
    if norm:
        if q is None or (k is None) != (dk is None):
            raise ValueError("norms need q and k")
        _heads(q, "q", dq, dq.shape)
        if k is not None:
            _heads(k, "k", dq, dk.shape)
    else:
        q = k = None
    own_q = own_k = ()
    if out_q is not None or out_k is not None:
        own_q = [t for t in (dq, q) if t is not None]
        own_k = [t for t in (dk, k) if t is not None]
    if out_q is None:
        out_q = _empty(m, hq, d, dq)
    else:
        _heads(out_q, "out_q", dq, dq.shape)
        _check_out(out_q, "out_q", own_q, own_k)
    if dk is None:
        if out_k is not None:
            raise ValueError("out_k needs dk")
    elif out_k is None:
        out_k = _empty(m, hk, d, dk)
    else:
        _heads(out_k, "out_k", dq, dk.shape)
        _check_out(out_k, "out_k", own_k, [*own_q, out_q])
    dw_q = dw_k = work = None
    need = 0
    if norm:
        dw_q = torch.empty_like(w_q)
        dw_k = None if dk is None else torch.empty_like(w_k)
        need = _bwd_workspace_bytes(m, hq, hk, d, dq.get_device())
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dq.device)
        else:
            workspace = _workspace_for(need, workspace, dq)
        work = workspace.data_ptr()
    _run(dq.get_device(), _lib.load().nf4s_rotary_bwd, dq.data_ptr(), _ptr(dk), _ptr(q), _ptr(k),
         int(dq.dtype == torch.bfloat16), m, hq, hk, d,
         _TWELVE(*dq.stride()[:2], *_pair(dk), *_pair(q), *_pair(k), *out_q.stride()[:2],
                 *_pair(out_k)), _ptr(w_q), _ptr(w_k), float(eps), positions.data_ptr(),
         rope.turns.data_ptr(), 2 * rope.turns.shape[0], int(rope.interleaved),
         float(rope.scale), out_q.data_ptr(), _ptr(out_k), _ptr(dw_q), _ptr(dw_k), work, need,
         _stream_ptr(dq))
    return RotaryGrad(out_q, out_k, dw_q, dw_k)
