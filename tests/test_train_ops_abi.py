"""Argument checks of the norms around a block, the 8-bit checkpoints and the
loss head through the C ABI, all refused before any launch (CPU only: the
pointers are dummies)."""
import ctypes

import pytest

from aethelstream_amd import _lib

INVALID = _lib.NF4S_ERR_INVALID_ARGUMENT
SHAPE = _lib.NF4S_ERR_UNSUPPORTED_SHAPE
ALIGN = _lib.NF4S_ERR_MISALIGNED
P = 0x1000


def _norm_fwd(**kw):
    a = dict(h=P, res=P, w_pre=P, w_post=P, gate=P, alpha=1.0, m=4, d=64, eps=1e-6, res_out=P, y=P,
             rms_pre=P, rms_post=P, stream=None)
    a.update(kw)
    return _lib.load().nf4s_block_norm_fwd(*a.values())


def _norm_bwd(**kw):
    a = dict(dy=P, dres=P, res=P, codes=None, scales=None, rms_pre=P, w_pre=P, h=P, rms_post=P,
             w_post=P, gate=P, alpha=1.0, m=4, d=64, dres_out=P, dh=P, dw_pre=P, dw_post=P, dgate=P,
             workspace=P, bytes=1 << 30, stream=None)
    a.update(kw)
    return _lib.load().nf4s_block_norm_bwd(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(m=-1), INVALID), (dict(d=0), INVALID), (dict(d=62), SHAPE), (dict(d=32772), SHAPE),
    (dict(m=1 << 40), SHAPE), (dict(h=None), INVALID), (dict(res=None), INVALID),
    (dict(w_pre=None), INVALID), (dict(rms_post=None), INVALID), (dict(y=None), INVALID),
    (dict(res=P + 8), ALIGN), (dict(h=P + 4), ALIGN), (dict(gate=P + 4), ALIGN)])
def test_block_norm_forward(kw, status):
    assert _norm_fwd(**kw) == status
    assert _lib.load().nf4s_last_error_message()


@pytest.mark.parametrize("kw,status", [
    (dict(m=-1), INVALID), (dict(d=0), INVALID), (dict(d=62), SHAPE), (dict(d=32772), SHAPE),
    (dict(dw_pre=None), INVALID), (dict(dw_post=None), INVALID), (dict(dgate=None), INVALID),
    (dict(w_post=None), INVALID), (dict(dy=None), INVALID), (dict(res=None), INVALID),
    (dict(codes=P, scales=P), INVALID), (dict(res=None, codes=P), INVALID),
    (dict(dh=None), INVALID), (dict(h=None, dh=None), INVALID), (dict(rms_post=None), INVALID),
    (dict(workspace=None), INVALID), (dict(bytes=16), INVALID), (dict(workspace=P + 8), ALIGN),
    (dict(dres=P + 8), ALIGN), (dict(dw_pre=P + 4), ALIGN), (dict(dy=P + 4), ALIGN)])
def test_block_norm_backward(kw, status):
    assert _norm_bwd(**kw) == status
    assert _lib.load().nf4s_last_error_message()


def test_checkpoints():
    lib = _lib.load()
    enc, dec, nrm = lib.nf4s_ckpt8_encode, lib.nf4s_ckpt8_decode, lib.nf4s_ckpt8_decode_norm
    for m, d, status in ((-1, 64, INVALID), (4, 0, INVALID), (4, 62, SHAPE),
                         (1 << 40, 128, SHAPE), (1 << 62, 1 << 31, SHAPE), (4, 1 << 40, SHAPE)):
        assert enc(P, 0, m, d, P, P, None) == status
        assert dec(P, P, m, d, P, 0, None) == status
        assert nrm(P, P, P, m, d, 1e-6, P, P, P, None) == status
    assert nrm(P, P, P, 4, 32772, 1e-6, P, P, P, None) == SHAPE
    assert enc(None, 0, 4, 64, P, P, None) == INVALID
    assert enc(P + 8, 0, 4, 64, P, P, None) == ALIGN
    assert enc(P + 4, 1, 4, 64, P, P, None) == ALIGN
    assert dec(P, P, 4, 64, None, 0, None) == INVALID
    assert dec(P + 2, P, 4, 64, P, 0, None) == ALIGN
    assert nrm(P, P, None, 4, 64, 1e-6, P, P, P, None) == INVALID
    assert nrm(P, P, P + 4, 4, 64, 1e-6, P, P, P, None) == ALIGN
    assert enc(None, 0, 0, 64, None, None, None) == 0
    assert dec(None, None, 0, 64, None, 0, None) == 0


def test_loss_head():
    lib = _lib.load()
    big = 1 << 40

    def fwd(x=P, w=P, t=P, m=4, v=32, d=64, loss=P, lse=P, work=P, size=big):
        return lib.nf4s_linear_ce_fwd(x, w, t, m, v, d, -100, loss, lse, work, size, None)

    def bwd(x=P, w=P, t=P, lse=P, dl=P, m=4, v=32, d=64, dx=P, dw=P, f32=0, acc=0, work=P,
            size=big):
        return lib.nf4s_linear_ce_bwd(x, w, t, lse, dl, m, v, d, -100, dx, dw, f32, acc, work,
                                      size, None)

    for f in (fwd, bwd):
        assert f(m=-1) == INVALID and f(v=0) == INVALID and f(d=0) == INVALID
        assert f(d=60) == SHAPE and f(v=1 << 29) == SHAPE and f(m=1 << 25) == SHAPE
        assert f(d=1 << 21) == SHAPE and f(m=1 << 24, v=1 << 28) == SHAPE
        assert f(x=None) == INVALID and f(w=None) == INVALID and f(t=None) == INVALID
        assert f(x=P + 8) == ALIGN and f(w=P + 2) == ALIGN and f(t=P + 4) == ALIGN
        assert f(work=None) == INVALID and f(size=16) == INVALID and f(work=P + 4) == ALIGN
    assert fwd(loss=None) == INVALID and fwd(lse=P + 2) == ALIGN
    assert bwd(dx=None) == INVALID and bwd(dw=None) == INVALID and bwd(dw=P + 8) == ALIGN
    assert bwd(acc=1) == INVALID
    assert b"fp32 only" in lib.nf4s_last_error_message()
    assert lib.nf4s_linear_ce_fwd(None, P, None, 0, 32, 64, -100, None, None, None, 0, None) == 0


def test_workspace_queries():
    lib = _lib.load()
    out = ctypes.c_int64(-1)
    q = lib.nf4s_linear_ce_workspace_size
    assert q(4, 32, 64, 0, None) == INVALID
    assert q(4, 32, 60, 0, ctypes.byref(out)) == SHAPE and out.value == 0
    assert q(0, 32, 64, 1, ctypes.byref(out)) == 0 and out.value == 0
    # Far less than the logits.
    for m, v, d in ((4096, 128000, 8192), (65536, 32000, 4096)):
        assert q(m, v, d, 0, ctypes.byref(out)) == 0 and 0 < out.value < m * v // 8
    assert q(4096, 128000, 8192, 1, ctypes.byref(out)) == 0
    assert out.value <= (256 << 20) + 4096 * 8192 * 4 + 16
    q = lib.nf4s_block_norm_bwd_workspace_size
    assert q(4, 64, None) == INVALID and q(4, 62, ctypes.byref(out)) == SHAPE
    assert q(0, 64, ctypes.byref(out)) == 0 and out.value == 0
