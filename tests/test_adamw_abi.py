"""Argument checks of the AdamW step through the C ABI, all refused before any launch
(CPU only: the pointers are dummies), and its coefficients."""
import ctypes
import os
import shutil
import subprocess

import pytest

from aethelstream_amd import _lib, build, optim

INVALID = _lib.NF4S_ERR_INVALID_ARGUMENT
SHAPE = _lib.NF4S_ERR_UNSUPPORTED_SHAPE
ALIGN = _lib.NF4S_ERR_MISALIGNED
P = 0x100000


def _ptrs(*v):
    return (ctypes.c_void_p * len(v))(*v)


def _step(params=(P, 2 * P), grads=(8 * P, 9 * P), copies=None, sizes=(1000, 5), types=(0, 0),
          count=2, m=16 * P, v=32 * P, ms=None, vs=None, hyper=(ctypes.c_float * 8)(), dev=None, scale=None):
    lists = [None if x is None else _ptrs(*x) for x in (params, grads, copies)]
    return _lib.load().nf4s_adamw_step(
        *lists, None if sizes is None else (ctypes.c_int64 * len(sizes))(*sizes),
        None if types is None else (ctypes.c_int32 * len(types))(*types), count, m, v, ms, vs, hyper,
        dev, scale, None)


@pytest.mark.parametrize("kw,status", [
    (dict(count=-1), INVALID), (dict(params=None), INVALID), (dict(grads=None), INVALID),
    (dict(sizes=None), INVALID), (dict(types=None), INVALID), (dict(hyper=None), INVALID),
    (dict(ms=P), INVALID), (dict(vs=P), INVALID), (dict(m=None), INVALID), (dict(v=None), INVALID),
    (dict(sizes=(-1, 5)), INVALID), (dict(types=(4, 0)), INVALID), (dict(types=(0, -1)), INVALID),
    (dict(params=(P, None)), INVALID), (dict(grads=(None, P)), INVALID),
    (dict(sizes=(1 << 40, 5)), SHAPE), (dict(sizes=((1 << 63) - 1, (1 << 63) - 1)), SHAPE),
    (dict(m=16 * P + 8), ALIGN), (dict(v=P + 4), ALIGN), (dict(ms=P + 2, vs=P), ALIGN),
    (dict(dev=P + 2), ALIGN), (dict(scale=P + 2), ALIGN), (dict(params=(P + 2, 2 * P)), ALIGN),
    (dict(types=(1, 0), params=(P + 1, 2 * P)), ALIGN), (dict(grads=(P, P + 2)), ALIGN),
    (dict(copies=(3 * P + 1, None)), ALIGN), (dict(copies=(3 * P, None), types=(1, 0)), INVALID),
    (dict(params=(P, P)), INVALID), (dict(params=(P, P + 3996)), INVALID),
    (dict(copies=(P + 100, None)), INVALID), (dict(copies=(3 * P, 3 * P + 1998)), INVALID),
    # Moments over each other or a parameter, a gradient in another tensor's parameter, in
    # its own shifted or of another type, in a copy, in the moments.
    (dict(v=16 * P), INVALID), (dict(v=P), INVALID), (dict(grads=(8 * P, P + 3984)), INVALID),
    (dict(grads=(P + 4, 9 * P)), INVALID), (dict(grads=(P, 9 * P), types=(2, 0)), INVALID),
    (dict(copies=(3 * P, None), grads=(8 * P, 3 * P)), INVALID),
    (dict(grads=(16 * P + 64, 9 * P)), INVALID)])
def test_refusals(kw, status):
    assert _step(**kw) == status
    assert _lib.load().nf4s_last_error_message()


def test_nothing_to_do():
    assert _step(count=0, params=None, grads=None, sizes=None, types=None) == 0
    assert _step(sizes=(0, 0), params=(None, None), grads=(None, None), m=None, v=None) == 0


def test_moments():
    f = _lib.load().nf4s_adamw_moments
    assert f(P, P, P, P, -1, P, P, None) == INVALID
    assert f(P, P, P, P, 1 << 33, P, P, None) == SHAPE
    assert f(None, P, P, P, 4, P, P, None) == INVALID
    assert f(P, P, P, P, 4, P, None, None) == INVALID
    assert f(P + 4, P, P, P, 4, P, P, None) == ALIGN
    assert f(P, P, P, P, 4, P + 8, P, None) == ALIGN
    assert f(None, None, None, None, 0, None, None, None) == 0


def test_coefficients():
    c = optim.coefficients(3, 0.1, (0.9, 0.99), 1e-8, 0.2)
    assert c == [0.9, 1 - 0.9, 0.99, 1 - 0.99, 1 - 0.1 * 0.2, 0.1 / (1 - 0.9 ** 3),
                 (1 - 0.99 ** 3) ** -0.5, 1e-8]
    for kw in (dict(step=0), dict(betas=(0.9, 1.0)), dict(lr=-1.0), dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            optim.coefficients(**{**dict(step=1, lr=0.1), **kw})


def test_state_layout():
    import torch
    state = optim.adamw_state([torch.zeros(3), torch.zeros(0), torch.zeros(2, 128),
                               torch.zeros(1)], bits=8)
    assert state.starts() == [0, 128, 128, 384] and state.m.numel() == 512
    assert state.m_scale.numel() == 4 and state.bits == 8


@pytest.mark.skipif(not (os.path.exists(build.HIPCC) or shutil.which(build.HIPCC)),
                    reason="needs hipcc")
def test_no_scratch_memory(tmp_path):
    out = str(tmp_path / "listing.s")
    subprocess.run([build.HIPCC, *build.HIP_FLAGS, "-S", "--offload-device-only",
                    os.path.join(build.CSRC, "adamw.hip"), "-o", out], check=True,
                   capture_output=True)
    with open(out) as f:
        text = f.read()
    kernels = text.count(".amdhsa_kernel ")
    assert kernels >= 13
    assert text.count(".amdhsa_private_segment_fixed_size 0\n") == kernels
