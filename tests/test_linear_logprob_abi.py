"""Argument checks of the log probabilities through the C ABI, all refused before any
launch, their workspaces, and the listing of their kernels (CPU only: the pointers are
dummies)."""
import ctypes
import os
import shutil
import subprocess

import pytest

import test_loss_listing as listing
from aethelstream_amd import _lib, build

INVALID = _lib.NF4S_ERR_INVALID_ARGUMENT
SHAPE = _lib.NF4S_ERR_UNSUPPORTED_SHAPE
ALIGN = _lib.NF4S_ERR_MISALIGNED
P = 0x1000
BIG = 1 << 42


def _fwd(x=P, w=P, t=P, m=4, v=32, d=64, k=3, logp=P, lse=P, ent=P, top=P, ids=P, logits=None,
         work=P, size=BIG):
    return _lib.load().nf4s_linear_logprob_fwd(x, w, t, m, v, d, k, -100, logp, lse, ent, top, ids,
                                               logits, work, size, None)


def _bwd(x=P, w=P, t=P, lse=P, ent=P, logits=None, da=P, dh=P, m=4, v=32, d=64, dx=P, dw=P, f32=0,
         acc=0, work=P, size=BIG):
    return _lib.load().nf4s_linear_logprob_bwd(x, w, t, lse, ent, logits, da, dh, m, v, d, -100,
                                               dx, dw, f32, acc, work, size, None)


def test_refusals():
    for f in (_fwd, _bwd):
        assert f(m=-1) == INVALID and f(v=0) == INVALID and f(d=0) == INVALID
        assert f(d=60) == SHAPE and f(v=1 << 29) == SHAPE and f(m=1 << 25) == SHAPE
        assert f(d=1 << 21) == SHAPE and f(m=1 << 24, v=1 << 28) == SHAPE
        assert f(x=None) == INVALID and f(w=None) == INVALID and f(t=None) == INVALID
        assert f(x=P + 8) == ALIGN and f(w=P + 2) == ALIGN and f(t=P + 4) == ALIGN
        assert f(work=None) == INVALID and f(size=16) == INVALID and f(work=P + 4) == ALIGN
        assert _lib.load().nf4s_last_error_message()
    assert _fwd(k=-1) == INVALID and _fwd(k=33, v=64) == SHAPE and _fwd(k=17, v=16) == SHAPE
    assert _fwd(logp=None) == INVALID and _fwd(lse=None) == INVALID and _fwd(ent=None) == INVALID
    assert _fwd(top=None) == INVALID and _fwd(ids=None) == INVALID
    assert _fwd(ent=P + 2) == ALIGN and _fwd(ids=P + 4) == ALIGN
    assert _bwd(dx=None) == INVALID and _bwd(dw=None) == INVALID and _bwd(dw=P + 8) == ALIGN
    assert _bwd(ent=None) == INVALID and _bwd(da=None) == INVALID and _bwd(dh=P + 2) == ALIGN
    assert _bwd(acc=1) == INVALID
    # Logits are kept of up to 16384 tokens, without alternatives.
    assert _fwd(logits=P) == SHAPE and _fwd(k=0, logits=P, m=16385) == SHAPE
    assert _fwd(k=0, logits=P + 8) == ALIGN
    assert _bwd(logits=P, m=16385) == SHAPE and _bwd(logits=P + 4) == ALIGN
    assert _fwd(m=0, x=None, t=None, logp=None, lse=None, ent=None, top=None, ids=None,
                work=None, size=0) == 0


def test_workspace():
    lib, out = _lib.load(), ctypes.c_int64(-1)
    q = lib.nf4s_linear_logprob_workspace_size
    assert q(4, 32, 64, 0, 0, None) == INVALID
    assert q(4, 32, 60, 0, 0, ctypes.byref(out)) == SHAPE and out.value == 0
    assert q(4, 32, 64, 33, 0, ctypes.byref(out)) == SHAPE
    assert q(0, 32, 64, 3, 0, ctypes.byref(out)) == 0 and out.value == 0
    for m, v, d in ((4096, 128000, 8192), (65536, 32000, 4096), (1, 128000, 4096)):
        assert q(m, v, d, 0, 0, ctypes.byref(out)) == 0 and 0 < out.value < m * v // 4
        without = out.value
        # Alternatives: a piece of the logits and the best ones so far.
        assert q(m, v, d, 8, 0, ctypes.byref(out)) == 0
        assert without < out.value < without + (270 << 20) + 100 * m
    f = lib.nf4s_linear_logprob_logits_size
    assert f(4, 32, 64, None) == INVALID and f(4, 32, 60, ctypes.byref(out)) == SHAPE
    for m, v, d in ((1, 40, 64), (77, 32000, 4096), (4096, 128000, 8192)):
        assert f(m, v, d, ctypes.byref(out)) == 0
        assert 4 * m * v <= out.value <= 4 * m * (v + 256)
    assert f(0, 32, 64, ctypes.byref(out)) == 0 and out.value == 0
    assert f(16385, 32, 64, ctypes.byref(out)) == 0 and out.value == 0
    assert q(4096, 128000, 8192, 0, 1, ctypes.byref(out)) == 0
    same = ctypes.c_int64(-1)
    lib.nf4s_linear_ce_workspace_size(4096, 128000, 8192, 1, ctypes.byref(same))
    assert out.value == same.value


@pytest.mark.skipif(not (os.path.exists(build.HIPCC) or shutil.which(build.HIPCC)),
                    reason="needs hipcc")
def test_listing(tmp_path):
    """No scratch memory, and the wide tiles' MFMAs keep their waits."""
    out = str(tmp_path / "listing.s")
    subprocess.run([build.HIPCC, *build.HIP_FLAGS, "-S", "--offload-device-only",
                    os.path.join(build.CSRC, "linear_logprob.hip"), "-o", out], check=True,
                   capture_output=True)
    with open(out) as f:
        text = f.read()
    kernels, tied = listing._kernels(text), 0
    for name, k in kernels.items():
        n, found = k.faults()
        tied += n > 0
        assert not found, (name, found[:5])
    assert tied == 4 and len(kernels) == 13, sorted(kernels)
    assert text.count(".amdhsa_private_segment_fixed_size 0\n") == len(kernels)
