"""The norms around a block where a workgroup takes several rows one after the
other: rows past the grid in both directions, with and without a block, from an
fp32 residual and from its checkpoint.  Formulas and tolerances are those of
test_block_norm_gpu.py.

Grids on 256 CUs.  Forward: 512 / t workgroups a CU for rows of t <= 512 threads
(four elements a chunk, four chunks a thread), one for longer rows.  Backward: two
chunks a thread up to 8192 columns, three up to 12288, eight beyond; 512 / t rows
side by side and 16 waves a CU."""
import pytest
import torch

import test_block_norm_gpu as bn
from aethelstream_amd import checkpoint, norm

pytestmark = pytest.mark.gpu


# Rows a workgroup: 5000 / 2048, 2500 / 1024, 1300 / 512, then m / 256.
@pytest.mark.parametrize("post,gate", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("m,d", [(5000, 512), (2500, 1028), (1300, 4096), (600, 8192), (600, 8196),
                                 (600, 12292), (777, 16384), (600, 16388)])
def test_forward(m, d, post, gate):
    print(m, d, post, gate, flush=True)
    s = bn._inputs(m, d, post, gate, seed=200)
    r = norm.block_norm_fwd(s["h"], s["res"], s["w_pre"], s["w_post"], s["gate"], bn.ALPHA)
    u, res, y, rms, rms_post = bn._forward64(s)
    bn._within(r.res, res, bn.U * (res.abs() + 64 * u.abs()) + bn.TINY)
    bn._within(r.rms_pre, rms[:, 0], 64 * bn.U * rms[:, 0])
    if post:
        bn._within(r.rms_post, rms_post[:, 0], 64 * bn.U * rms_post[:, 0])
    slack = 64 * bn.U * (res.abs() + u.abs()) / rms * s["w_pre"].double().abs()
    bn._within(r.y, y, 2.0 ** -8 * y.abs() + 2 * slack + bn.TINY)


ROWS = [(9000, 1024), (5003, 1028), (1500, 4096), (1100, 8192), (600, 8196), (801, 12288),
        (1100, 12292), (600, 16384), (600, 16388)]


def _backward(m, d, s, dres, bits8):
    dy = bn._randn((m, d), 220, 1e-3, torch.bfloat16)
    res = bn._randn((m, d), 222, 1.5)
    source = checkpoint.encode(res) if bits8 else res
    if bits8:
        res = checkpoint.decode(source)
    rms = bn._rms(res.double(), norm.EPS)[:, 0].float()
    post = s["w_post"] is not None
    rms_post = bn._rms(s["h"].double(), norm.EPS)[:, 0].float() if post else None
    r = norm.block_norm_bwd(dy, dres, source, rms, s["w_pre"], s["h"], rms_post, s["w_post"],
                            s["gate"], bn.ALPHA)
    want = bn._backward64(s, dy, torch.zeros_like(res) if dres is None else dres, res, rms,
                          rms_post)
    bn._check_backward(r, want, m)


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("post,gate", [(False, False), (True, True)])
@pytest.mark.parametrize("m,d", ROWS)
def test_backward(m, d, post, gate, bits8):
    print(m, d, post, gate, bits8, flush=True)
    s = bn._inputs(m, d, post, gate, seed=210)
    _backward(m, d, s, bn._randn((m, d), 221, 1e-3), bits8)


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("m,d", ROWS)
def test_backward_without_block(m, d, given, bits8):
    print(m, d, given, bits8, flush=True)
    s = dict(bn._inputs(m, d, False, False, seed=230), h=None)
    _backward(m, d, s, bn._randn((m, d), 221, 1e-3) if given else None, bits8)
