"""8-bit moments take beta1 and beta2 up to 0.95: beyond, a step changes them by less than
half the distance of two codes, which rounding to nearest drops.  Refused on the host
before any launch (CPU: the pointers are dummies); coefficients on the device are only
seen there, and leave NaN.

What holds at 0.95, against 32-bit moments, for normal gradients, where a step changes
sqrt(v) by a random part of it: a rounding is off by at most 2^-5 of the value, uniform
within half a code's distance, 0.013 of it in the rms over a binade.  The next step keeps
0.95 of that, so it adds up to 0.013 / sqrt(1 - 0.95^2) = 0.042 in the rms.  A single
value gets four times that, the mean over thousands (whose own spread is 0.0005) 0.02.
"""
import ctypes

import pytest
import torch

from aethelstream_amd import _lib, optim

INVALID = _lib.NF4S_ERR_INVALID_ARGUMENT
P = 0x100000


def _host_step(betas, bits8=True):
    hyper = (ctypes.c_float * 8)(*optim.coefficients(3, 1e-3, betas))
    lists = [(ctypes.c_void_p * 1)(a) for a in (P, 8 * P)]
    scales = (P * 3, P * 4) if bits8 else (None, None)
    # (Of the unknown type -1, so that what is not refused before is refused then.)
    return _lib.load().nf4s_adamw_step(*lists, None, (ctypes.c_int64 * 1)(1000),
                                       (ctypes.c_int32 * 1)(-1), 1, 16 * P, 32 * P, *scales, hyper,
                                       None, None, None)


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.9, 0.96), (0.99, 0.95), (0.951, 0.9)])
def test_refused_by_the_library(betas):
    assert _host_step(betas) == INVALID
    assert b"0.95" in _lib.load().nf4s_last_error_message()


@pytest.mark.parametrize("betas,bits8", [((0.95, 0.95), True), ((0.9, 0.95), True),
                                         ((0.0, 0.0), True), ((0.9, 0.999), False)])
def test_not_refused_by_the_library(betas, bits8):
    assert _host_step(betas, bits8) == INVALID
    assert b"unknown type" in _lib.load().nf4s_last_error_message()


@pytest.mark.gpu
def test_refused_by_the_step():
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    state = optim.adamw_state([p], bits=8)
    for kw in (dict(), dict(betas=(0.9, 0.999)), dict(betas=(0.96, 0.9))):
        with pytest.raises(ValueError, match="0.95"):
            optim.adamw_step([p], [g], state, 1, **kw)
    assert (p == 1).all() and not state.m.any() and not state.v_scale.any()
    optim.adamw_step([p], [g], state, 1, betas=(0.95, 0.95))
    optim.adamw_step([p.clone()], [g], optim.adamw_state([p]), 1)  # 32 bits: the default
    assert (p != 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.96, 0.95), (float("nan"), 0.9)])
def test_coefficients_on_the_device_leave_nan(betas):
    p, q = torch.ones(300, device="cuda"), torch.ones(5, device="cuda", dtype=torch.bfloat16)
    state = optim.adamw_state([p, q], bits=8)
    hyper = torch.tensor([betas[0], 0.1, betas[1], 0.1, 1.0, 1e-3, 1.0, 1e-8], device="cuda")
    optim.adamw_step([p, q], [p.clone(), q.clone()], state, 1, hyper=hyper)
    assert p.isnan().all() and q.isnan().all()
    assert state.m_scale.isnan().all() and state.v_scale.isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("change", [1.0, 2.0, 4.0, 0.5, 0.1])
def test_moments_follow_gradients_that_vary(change):
    """Blocks of 128 with one channel far louder than the others, whose gradients change
    by a factor after 200 steps: 400 steps later v is what 32 bits have."""
    g = torch.Generator(device="cuda").manual_seed(7)
    size = torch.exp(0.7 * torch.randn(64, 128, device="cuda", generator=g))
    size[:, 0] = 8 * size.amax(1)
    p = torch.zeros(64 * 128, device="cuda")
    q = p.clone()
    a, b = optim.adamw_state([p], bits=8), optim.adamw_state([q])
    total = torch.zeros(2, 64, 128, device="cuda", dtype=torch.float64)
    for t in range(600):
        if t == 200:
            size[:, 1:] *= change
        grad = (size * torch.randn(64, 128, device="cuda", generator=g)).view(-1)
        optim.adamw_step([p], [grad], a, t + 1, betas=(0.9, 0.95))
        optim.adamw_step([q], [grad], b, t + 1, betas=(0.9, 0.95))
        if t >= 400:
            for i, s in enumerate((a, b)):
                total[i] += optim.moments(s)[1].view(64, 128).double().sqrt()
    share = (total[0] / total[1])[:, 1:]
    assert abs(float(share.mean()) - 1) < 0.02
    assert float((share - 1).abs().max()) < 4 * 0.042
