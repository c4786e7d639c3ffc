"""Loss head, norms around a block and 8-bit checkpoints on tensors past 2^31
elements, where a 32-bit offset would wrap: the first and last rows against the
plain forms, and the sums over rows with every other row's share zero.  The
tolerances are those of the operators' own tests."""
import dataclasses

import numpy as np
import pytest
import torch

import test_block_norm_gpu as bn
import test_ckpt8_gpu as c8
import test_linear_ce_gpu as ce
from aethelstream_amd import checkpoint, loss, norm

pytestmark = pytest.mark.gpu

ROWS, D = 65600, 32768  # 2^31 + 2 M elements
EDGE = 8


def _edges():
    return torch.cat([torch.arange(EDGE, device="cuda"),
                      torch.arange(ROWS - EDGE, ROWS, device="cuda")])


def test_block_norm_rows():
    print("forward", ROWS, D, flush=True)
    e = _edges()
    s = bn._inputs(ROWS, D, True, True, seed=50)
    r = norm.block_norm_fwd(s["h"], s["res"], s["w_pre"], s["w_post"], s["gate"], bn.ALPHA)
    few = dict(s, h=s["h"][e], res=s["res"][e])
    small = norm.block_norm_fwd(few["h"], few["res"], s["w_pre"], s["w_post"], s["gate"], bn.ALPHA)
    u, res, y, rms, rms_post = bn._forward64(few)
    bn._within(r.res[e], res, bn.U * (res.abs() + 64 * u.abs()) + bn.TINY)
    bn._within(r.rms_pre[e], rms[:, 0], 64 * bn.U * rms[:, 0])
    bn._within(r.rms_post[e], rms_post[:, 0], 64 * bn.U * rms_post[:, 0])
    for name in ("res", "y", "rms_pre", "rms_post"):
        assert torch.equal(getattr(r, name)[e], getattr(small, name))

    print("backward", ROWS, D, flush=True)
    dy = torch.zeros(ROWS, D, dtype=torch.bfloat16, device="cuda")
    dres = torch.zeros(ROWS, D, device="cuda")
    dy[e] = bn._randn((2 * EDGE, D), 51, 1e-3, torch.bfloat16)
    dres[e] = bn._randn((2 * EDGE, D), 52, 1e-3)
    for source in (r.res, checkpoint.encode(r.res)):
        at = r.res if source is r.res else checkpoint.decode(source)
        g = norm.block_norm_bwd(dy, dres, source, r.rms_pre, s["w_pre"], s["h"], r.rms_post,
                                s["w_post"], s["gate"], bn.ALPHA)
        want = bn._backward64(few, dy[e], dres[e], at[e], r.rms_pre[e], r.rms_post[e])
        bn._check_backward(dataclasses.replace(g, dres=g.dres[e], dh=g.dh[e]), want, ROWS)
        # Rows without a gradient give exactly none.
        assert not g.dres[EDGE:-EDGE].any() and not g.dh[EDGE:-EDGE].any()


def test_checkpoint_rows():
    print("checkpoint", ROWS, D, flush=True)
    e = _edges()
    x = c8._randn((ROWS, D), 53, 2.0)
    c = checkpoint.encode(x)
    codes, scales = c8._reference(x[e])
    assert np.array_equal(c.codes[e].cpu().numpy(), codes)
    assert np.array_equal(c.scales[e].cpu().numpy(), scales)
    del x
    values = torch.from_numpy(codes.astype(np.float32) * np.repeat(scales, 128, 1)).cuda()
    assert torch.equal(checkpoint.decode(c)[e], values)
    w = 1 + c8._randn((D,), 54, 0.1)
    x, y, rms = checkpoint.decode_norm(c, w)
    small = checkpoint.decode_norm(checkpoint.Checkpoint8(c.codes[e], c.scales[e]), w)
    assert torch.equal(x[e], values)
    assert torch.equal(y[e], small[1]) and torch.equal(rms[e], small[2])


def test_loss_of_many_tokens():
    """x past 2^31 elements; all tokens but the first and last are ignored in the sums."""
    print("tokens", ROWS, 40, D, flush=True)
    e = _edges()
    x, w, t, dl = ce._inputs(ROWS, 40, D, seed=55, skip=0.0)
    t[EDGE:-EDGE] = loss.IGNORE_INDEX
    out, lse = loss.linear_cross_entropy(x, w, t)
    ce._check_forward(x[e], w, t[e], (out[e], lse[e]))
    assert not out[EDGE:-EDGE].any()
    dx, dw = loss.linear_cross_entropy_bwd(x, w, t, lse, dl)
    ce._check_backward(x[e], w, t[e], dl[e], lse[e], dx[e], dw)
    assert not dx[EDGE:-EDGE].any()


def test_loss_of_a_large_vocabulary():
    """w and dw past 2^31 elements, targets at both ends."""
    print("vocabulary", 40, ROWS, D, flush=True)
    x, w, t, dl = ce._inputs(40, ROWS, D, seed=56)
    t[:4] = torch.tensor([0, ROWS - 1, ROWS - 2, 1], device="cuda")
    out, lse = loss.linear_cross_entropy(x, w, t)
    ce._check_forward(x, w, t, (out, lse))
    dx, dw = loss.linear_cross_entropy_bwd(x, w, t, lse, dl)
    ce._check_backward(x, w, t, dl, lse, dx, dw)
