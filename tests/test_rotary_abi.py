"""Argument checks of the rotation through the C ABI, all refused before any launch
(CPU only: the pointers are dummies), and its angles against 64-bit arithmetic."""
import ctypes
import math
import os
import shutil
import subprocess

import pytest

from aethelstream_amd import _lib, build, rotary

INVALID = _lib.NF4S_ERR_INVALID_ARGUMENT
SHAPE = _lib.NF4S_ERR_UNSUPPORTED_SHAPE
ALIGN = _lib.NF4S_ERR_MISALIGNED
P = 0x1000
STRIDES = (ctypes.c_int64 * 12)(*([1024, 64] * 6))


def _fwd(**kw):
    a = dict(q=P, k=P, is_bf16=1, m=4, hq=4, hk=2, d=64, strides=STRIDES, w_q=P, w_k=P, eps=1e-6,
             positions=P, turns=P, rot=64, interleaved=0, scale=1.0, q_out=P, k_out=P, stream=None)
    a.update(kw)
    return _lib.load().nf4s_rotary_fwd(*a.values())


def _bwd(**kw):
    a = dict(dq=P, dk=P, q=P, k=P, is_bf16=1, m=4, hq=4, hk=2, d=64, strides=STRIDES, w_q=P, w_k=P,
             eps=1e-6, positions=P, turns=P, rot=64, interleaved=0, scale=1.0, dq_out=P, dk_out=P,
             dw_q=P, dw_k=P, workspace=P, bytes=1 << 30, stream=None)
    a.update(kw)
    return _lib.load().nf4s_rotary_bwd(*a.values())


COMMON = [
    (dict(m=-1), INVALID), (dict(hq=0), INVALID), (dict(hk=-1), INVALID), (dict(d=0), INVALID),
    (dict(rot=0), INVALID), (dict(d=63, rot=2), SHAPE), (dict(rot=63), SHAPE),
    (dict(rot=66), SHAPE), (dict(d=1026), SHAPE), (dict(hq=4097), SHAPE), (dict(hk=4097), SHAPE),
    (dict(m=(1 << 32) + 1), SHAPE), (dict(q=None), INVALID), (dict(k=None), INVALID),
    (dict(strides=None), INVALID), (dict(positions=None), INVALID), (dict(turns=None), INVALID),
    (dict(w_q=None), INVALID), (dict(w_k=None), INVALID), (dict(q=P + 1), ALIGN),
    (dict(is_bf16=0, k=P + 2), ALIGN), (dict(positions=P + 4), ALIGN), (dict(turns=P + 4), ALIGN),
    (dict(w_q=P + 2), ALIGN)]


@pytest.mark.parametrize("kw,status", COMMON + [
    (dict(q_out=None), INVALID), (dict(k_out=None), INVALID), (dict(q_out=P + 1), ALIGN)])
def test_forward(kw, status):
    assert _fwd(**kw) == status
    assert _lib.load().nf4s_last_error_message()


@pytest.mark.parametrize("kw,status", COMMON + [
    (dict(dq=None), INVALID), (dict(dk=None), INVALID), (dict(dq_out=None), INVALID),
    (dict(dk_out=None), INVALID), (dict(dw_q=None), INVALID), (dict(dw_k=None), INVALID),
    (dict(w_q=None, w_k=None), INVALID), (dict(workspace=None), INVALID), (dict(bytes=16), INVALID),
    (dict(workspace=P + 2), ALIGN), (dict(dk=P + 1), ALIGN), (dict(dw_q=P + 2), ALIGN)])
def test_backward(kw, status):
    assert _bwd(**kw) == status
    assert _lib.load().nf4s_last_error_message()


def test_no_tokens_and_workspace():
    assert _fwd(m=0, q=None, k=None, q_out=None, k_out=None, positions=None, strides=None) == 0
    assert _bwd(m=0, w_q=None, w_k=None, dw_q=None, dw_k=None, dq=None, dk=None) == 0
    lib, out = _lib.load(), ctypes.c_int64(-1)
    f = lib.nf4s_rotary_bwd_workspace_size
    assert f(4, 4, 2, 64, None) == INVALID
    assert f(4, 4, 2, 63, ctypes.byref(out)) == SHAPE and out.value == 0
    assert f(0, 4, 2, 64, ctypes.byref(out)) == 0 and out.value == 0
    assert f(1, 4, 2, 64, ctypes.byref(out)) == 0 and out.value == 6 * 64 * 4
    # Bounded by the workgroups, not by the rows.
    assert f(1 << 32, 64, 8, 128, ctypes.byref(out)) == 0 and out.value == 1025 * 128 * 4


def test_frequencies():
    f, scale = rotary.frequencies(8, base=100.0)
    assert scale == 1.0 and f == [100.0 ** (-i / 4) for i in range(4)]
    g, scale = rotary.frequencies(8, base=100.0, factor=2.0)
    assert scale == 1.0 and g == [v / 2 for v in f]
    # Pairs that turn 32 times in the trained length keep their frequency, those that
    # turn once are divided, the others lie between.
    f, _ = rotary.frequencies(128)
    g, scale = rotary.frequencies(128, factor=4.0, trained=8192)
    assert scale == pytest.approx(0.1 * math.log(4) + 1)
    for a, b in zip(f, g):
        turns = 8192 * a / (2 * math.pi)
        assert a / 4 * (1 - 1e-12) <= b <= a * (1 + 1e-12)
        if turns > 34:
            assert b == a
        if turns < 0.9:
            assert b == pytest.approx(a / 4)
    for kw in (dict(rot=0), dict(rot=7), dict(rot=8, factor=0.5), dict(rot=8, base=0.0),
               dict(rot=8, factor=2.0, trained=0), dict(rot=8, factor=2.0, trained=9, slow=40.0)):
        with pytest.raises(ValueError):
            rotary.frequencies(**kw)


def test_turns():
    """Units of 2^-64 turns of any frequency, negative and above a turn among them."""
    radians = [1.0, 0.25, -0.25, 3.5, 100.0, 1e-7, math.pi, 0.0]
    rope = rotary.Rotary.from_frequencies(radians, device="cpu")
    for v, t in zip(radians, rope.turns.tolist()):
        want = v / (2 * math.pi) % 1.0
        assert abs((t % (1 << 64)) * 2.0 ** -64 - want) <= 2.0 ** -52 * max(1.0, abs(v))
    with pytest.raises(ValueError):
        rotary.Rotary.from_frequencies([float("nan")], device="cpu")


def test_places_of_outputs():
    """An output is one of its own inputs or lies apart from each of them, and from the
    others; parts of one row lie apart."""
    import torch
    flat = torch.zeros(4 * 6 * 8 + 100)
    rows = flat[:192].view(4, 6, 8)
    q, k, rest = rows[:, :3], rows[:, 3:5], rows[:, 5:]
    rotary._check_out(q, "out", [q], [k, rest])
    rotary._check_out(k, "out", [], [q, rest])
    rotary._check_out(q, "out", [q, q], [k])
    shifted = flat[4:196].view(4, 6, 8)[:, :3]
    for own, others in (([], [q]), ([shifted], []), ([q, shifted], []), ([shifted, q], []),
                        ([q], [shifted]), ([rows], [])):
        with pytest.raises(ValueError):
            rotary._check_out(q, "out", own, others)
    with pytest.raises(ValueError):
        rotary._check_out(flat[:8].expand(4, 3, 8), "out", [], [])


def test_refuses_host_tensors():
    import torch
    q = torch.zeros(2, 2, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        rotary.apply(q, None, torch.zeros(2, dtype=torch.int64),
                     rotary.Rotary(torch.zeros(4, dtype=torch.int64)))


@pytest.mark.skipif(not (os.path.exists(build.HIPCC) or shutil.which(build.HIPCC)),
                    reason="needs hipcc")
def test_no_scratch_memory(tmp_path):
    out = str(tmp_path / "listing.s")
    subprocess.run([build.HIPCC, *build.HIP_FLAGS, "-S", "--offload-device-only",
                    os.path.join(build.CSRC, "rotary.hip"), "-o", out], check=True,
                   capture_output=True)
    with open(out) as f:
        text = f.read()
    kernels = text.count(".amdhsa_kernel ")
    assert kernels >= 13
    assert text.count(".amdhsa_private_segment_fixed_size 0\n") == kernels
