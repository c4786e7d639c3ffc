"""8-bit moments whose gradients are zero, or become zero, beside others of their block:
m falls with every step until it is zero, as rounding to nearest alone would hold it at
one of its lowest codes, and the parameter would go on for good.  Codes bit for bit
against the same fp32 operations in numpy, and the way of the parameters against 32
bits."""
import numpy as np
import pytest
import torch

import test_adamw_gpu as ad
from aethelstream_amd import optim

pytestmark = pytest.mark.gpu


def _np_codes(state, grads, step, scale=1.0):
    """What test_adamw_gpu._np_step has, but that the code of m of a zero gradient is one
    lower where it would stand for no less than before."""
    want = list(ad._np_step(state, grads, step, scale))
    old = np.abs(ad._np_moments(state)[0])
    g = np.ones_like(old)
    for a, n, t in zip(state.starts(), state.sizes, grads):
        g[a:a + n] = t.float().cpu().numpy() * np.float32(scale)
    mag = np.abs(want[0].astype(np.int32))
    with np.errstate(all="ignore"):
        now = ad._np_value(mag, want[2], 3)
        held = (g == 0) & (mag > 0) & (now >= old)
    mag = mag - held
    want[0] = np.where(want[0] < 0, -mag, mag).astype(np.int8)
    return want, int(held.sum())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", [[129, 4096, 1, 77], [70000]])
def test_codes(dtype, sizes):
    """Every third element's gradients are small, then zero (of either sign); in some
    steps all are.  Where m is of the lowest codes the rule decides in several steps of
    each."""
    ps = [ad._randn((n,), i, 0.02, dtype) for i, n in enumerate(sizes)]
    state = optim.adamw_state(ps, bits=8)
    total = 0
    for step in range(1, 41):
        gs = [ad._randn((n,), 100 * step + i, 1.0, dtype) for i, n in enumerate(sizes)]
        for g in gs:
            if step % 10 == 5:
                g.zero_()
            elif step > 3:
                g[::3] = 0.0 if step % 2 else -0.0
            else:
                g[::3] *= 1e-4
        want, held = _np_codes(state, gs, step)
        total += held
        optim.adamw_step(ps, gs, state, step, ad.LR, ad.BETAS, ad.EPS, ad.WD)
        ad._check_codes(state, want)
    assert total > sum(sizes) // 3
    assert all(p.isfinite().all() for p in ps)


def test_scaled_to_zero():
    """A factor of zero makes every gradient one of zero."""
    p, g = ad._randn((3000,), 1, 0.02), ad._randn((3000,), 2)
    state = optim.adamw_state([p], bits=8)
    optim.adamw_step([p], [g], state, 1, ad.LR, ad.BETAS, ad.EPS, ad.WD)
    for step in range(2, 12):
        want, _ = _np_codes(state, [g], step, 0.0)
        optim.adamw_step([p], [g], state, step, ad.LR, ad.BETAS, ad.EPS, ad.WD,
                         grad_scale=torch.zeros(1, device="cuda"))
        ad._check_codes(state, want)


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.95, 0.95), (0.9, 0.9)])
@pytest.mark.parametrize("kind", ["normal", "sign", "constant"])
def test_parameters_come_to_rest(betas, kind):
    """Every fourth element of a block has no gradient from step 101 on: 300 steps later
    none of them moves by 1e-3 of lr a step on average.  (In 32 bits, beta1^t /
    beta2^(t / 2) of what it was: below 1e-3 at 0.95, and far below at the others.)"""
    gen = torch.Generator(device="cuda").manual_seed(5)
    size = torch.exp(0.7 * torch.randn(48, 128, device="cuda", generator=gen))
    p = torch.zeros(48 * 128, device="cuda")
    state = optim.adamw_state([p], bits=8)
    lr, steps, at = 1e-3, 700, None
    for t in range(1, steps + 1):
        g = torch.randn(48, 128, device="cuda", generator=gen)
        g = size * (g if kind == "normal" else g.sign() if kind == "sign" else 1.0)
        if t > 100:
            g[:, ::4] = 0
        optim.adamw_step([p], [g.view(-1)], state, t, lr, betas)
        if t == 400:
            at = p.clone()
    moved = (p - at).view(48, 128).double().abs() / lr / (steps - 400)
    assert float(moved[:, ::4].max()) < 1e-3
    # The others go on.
    assert float(moved[:, 1::4].mean()) > 1e-2
