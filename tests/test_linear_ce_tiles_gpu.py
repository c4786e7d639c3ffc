"""The loss head where its launches take other tiles than the small shapes of
test_linear_ce_gpu.py: 128 x 256 tiles of logits, alone and beside others, lengths
that end inside a step of 64, partial last columns; several pieces of the
vocabulary, with targets on both sides of a piece's end; fp32 dw that accumulates.
Formulas and tolerances are those of that file.  (Tiles: the rules' choice on 256
CUs.)"""
import pytest
import torch

import test_linear_ce_gpu as ce
from aethelstream_amd import loss

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,v,d", [
    (77, 50021, 1032), (256, 32001, 1000),  # 128 x 256
    (66, 69293, 1992),   # 128 x 256, then 64 x 128
    (275, 53493, 1280),  # 256 x 256, then 128 x 256
    (208, 66047, 952), (777, 33001, 1032),  # 256 x 256, then 64 x 128
    (77, 32003, 4096)])  # 64 x 128
def test_tiles(m, v, d):
    print(m, v, d, flush=True)
    x, w, t, dl = ce._inputs(m, v, d, seed=m)
    t[:3] = torch.tensor([0, v - 1, v - 2], device="cuda")
    out, lse = loss.linear_cross_entropy(x, w, t)
    ce._check_forward(x, w, t, (out, lse))
    dx, dw = loss.linear_cross_entropy_bwd(x, w, t, lse, dl)
    ce._check_backward(x, w, t, dl, lse, dx, dw)


def _piece(m, v):
    """Columns of a piece: G in bf16 within 256 MB and 2^20 columns, in 256s."""
    most = max(256, min((256 << 20) // (2 * m) // 256 * 256, 1 << 20))
    pieces = -(-v // most)
    return min(v, -(-(-(-v // pieces)) // 256) * 256)


def _check_pieces(x, w, t, dl, lse, dx, dw, before, cols):
    """dx, and rows ``cols`` of dw (added to ``before``), as _check_backward."""
    z, _, _ = ce._forward64(x, w, t)
    rel = (ce._logit_error(x, w) + ce.U * (64 + 4 * lse.double().abs()))[:, None]
    p = torch.exp(z - lse.double()[:, None])
    del z
    hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0)
    scale = ((t != loss.IGNORE_INDEX).double() * dl.double())[:, None]
    g = (p - hot) * scale
    off = (2.0 ** -8 + 4 * ce.U) * g.abs() + (p * rel + ce.U * hot) * scale.abs()
    del p, hot
    wide = w.double()
    want = g @ wide
    wide = wide.abs_()
    bound = off @ wide + (2.0 ** -8 + 2 * ce.U * x.shape[1]) * want.abs() \
        + 64 * ce.U * (g.abs() @ wide) + 1e-30
    assert ((dx.double() - want).abs() <= bound).all()
    g, off = g[:, cols].t(), off[:, cols].t()
    want = g @ x.double() + before[cols].double()
    bound = off @ x.double().abs() + 64 * ce.U * (g.abs() @ x.double().abs()) \
        + 2 * ce.U * want.abs() + 1e-30
    assert ((dw[cols].double() - want).abs() <= bound).all()


# Few tokens: pieces of 2^20 columns at most, dx in tiles of 64, 128 and 128 rows,
# dw in 128 x 128 and, past 128 tokens, 256 x 256 tiles.
@pytest.mark.parametrize("m,v,d", [(5, 1100003, 2048), (100, 1100003, 64), (300, 1000003, 64),
                                   (2500, 60001, 520)])
def test_pieces_accumulate(m, v, d):
    print(m, v, d, flush=True)
    piece = _piece(m, v)
    assert piece < v
    x, w, t, dl = ce._inputs(m, v, d, seed=m + 1, skip=0.0)
    edge = torch.tensor([0, piece - 1, piece, v - 1], device="cuda")
    t[:4] = edge
    t[4] = loss.IGNORE_INDEX
    _, lse = loss.linear_cross_entropy(x, w, t)
    cols = torch.cat([t[t >= 0], torch.arange(piece - 40, piece + 40, device="cuda"),
                      torch.arange(v - 300, v, device="cuda")])
    before = ce._randn((v, d), m + 2, 0.1, torch.float32)
    dw = before.clone()
    dx, same = loss.linear_cross_entropy_bwd(x, w, t, lse, dl, dw=dw, accumulate=True)
    assert same is dw
    _check_pieces(x, w, t, dl, lse, dx, dw, before, cols)
    # Stored, then rounded: the same products.
    dx2, stored = loss.linear_cross_entropy_bwd(x, w, t, lse, dl, dw=torch.empty_like(before))
    dx3, rounded = loss.linear_cross_entropy_bwd(x, w, t, lse, dl)
    assert torch.equal(dx, dx2) and torch.equal(dx, dx3)
    assert torch.equal(before + stored, dw) and torch.equal(stored.to(torch.bfloat16), rounded)


@pytest.mark.parametrize("m,v,d", [(1, 3001, 520), (77, 3001, 520), (128, 1000, 72),
                                   (129, 1000, 72), (600, 2000, 264)])
def test_accumulate_micro_batches(m, v, d):
    """Two micro-batches into one dw: each adds its own sum, rounded once."""
    total = torch.zeros(v, d, device="cuda")
    want = torch.zeros(v, d, device="cuda")
    for seed in (20, 40):
        x, w, t, dl = ce._inputs(m, v, d, seed=seed)
        _, lse = loss.linear_cross_entropy(x, w, t)
        before = total.clone()
        dx, _ = loss.linear_cross_entropy_bwd(x, w, t, lse, dl, dw=total, accumulate=True)
        ce._check_backward(x, w, t, dl, lse, dx, total, accumulated=before)
        one = torch.empty_like(total)
        loss.linear_cross_entropy_bwd(x, w, t, lse, dl, dw=one)
        want += one
        assert torch.equal(want, total)
