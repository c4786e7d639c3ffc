"""Kept logits of the log probabilities: they belong to one shape, and the gradients take
them piece by piece of the vocabulary."""
import pytest
import torch

import test_linear_ce_gpu as ce
import test_linear_logprob_gpu as lp
import test_linear_logprob_plan as plan
from aethelstream_amd import loss

pytestmark = pytest.mark.gpu


def _kept(m, v, d, seed=1):
    x, w, t, da = ce._inputs(m, v, d, seed=seed)
    return x, w, t, da, loss.linear_log_probs(x, w, t, keep_logits=True)


def test_of_another_shape():
    """Logits of as many elements, but of another vocabulary or another reduction."""
    m, d = 40, 64
    x, w, t, da, r = _kept(m, 100, d)
    x2, w2, t2, da2, s = _kept(m, 101, d)
    x3, w3, t3, da3, u = _kept(m, 100, 2 * d)
    assert r.logits.numel() == s.logits.numel() == u.logits.numel()
    for a in ((x, w, t, s), (x2, w2, t2, r), (x, w, t, u), (x3, w3, t3, r)):
        with pytest.raises(ValueError, match="another head"):
            loss.linear_log_probs_bwd(*a, da)
    # Logits of no known shape.
    with pytest.raises(ValueError, match="another head"):
        loss.linear_log_probs_bwd(
            x, w, t, loss.LogProbs(r.logp, r.entropy, r.lse, None, None, r.logits), da)
    dx, dw = loss.linear_log_probs_bwd(x, w, t, r, da)
    assert r.shape == (m, 100, d) and dx.isfinite().all() and dw.isfinite().all()
    # A result of its parts, with the logits' shape or without the logits.
    for parts in ((r.logits, r.shape), ()):
        got = loss.linear_log_probs_bwd(
            x, w, t, loss.LogProbs(r.logp, r.entropy, r.lse, None, None, *parts), da)
        assert torch.equal(got[0], dx) and torch.equal(got[1], dw)


@pytest.mark.parametrize("m,v,d,first", plan.PIECES)
def test_pieces_of_the_gradient(m, v, d, first):
    """Gradients from kept logits over several pieces, the last one shorter, are those
    from logits made again, bit for bit, and those of 64 bits for the tokens that have
    any; with targets on both sides of every border."""
    print(m, v, d, flush=True)
    assert loss.log_probs_workspace_bytes(m, v, d, backward=True) < 2 * m * v
    x, w, t, da, r = _kept(m, v, d, seed=m)
    piece = plan._up(-(-v // -(-v // ((1 << 28) // (2 * m) // 256 * 256))), 256)
    edges = [0, v - 1]
    for c in [*range(piece, v, piece), *([first] if first else [])]:
        edges += [c - 1, c]
    t[:len(edges)] = torch.tensor(edges, device="cuda")
    few = min(m, 300) // 2
    dh = ce._randn((m,), 9, 0.5, torch.float32)
    da[few:-few] = 0
    dh[few:-few] = 0
    rows = torch.cat([torch.arange(few, device="cuda"), torch.arange(m - few, m, device="cuda")])
    r = loss.linear_log_probs(x, w, t, keep_logits=True)
    s = loss.linear_log_probs(x, w, t, keep_logits=False)
    got = None
    for b in (None, dh):
        got = loss.linear_log_probs_bwd(x, w, t, r, da, b)
        want = loss.linear_log_probs_bwd(x, w, t, s, da, b)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert not got[0][few:-few].any()
    part = loss.LogProbs(r.logp[rows], r.entropy[rows], r.lse[rows], None, None)
    lp._check_forward(x[rows], w, t[rows], part)
    lp._check_backward(x[rows], w, t[rows], da[rows], dh[rows], part, got[0][rows], got[1])


def test_workspace_that_held_something_over_pieces():
    """G of the last, shorter piece lies where the one before was: NaN there first."""
    m, v, d, _ = plan.PIECES[0]
    x, w, t, da, r = _kept(m, v, d, seed=3)
    dh = ce._randn((m,), 9, 0.5, torch.float32)
    need = loss.log_probs_workspace_bytes(m, v, d, backward=True)
    want = loss.linear_log_probs_bwd(x, w, t, r, da, dh)
    work = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
    got = loss.linear_log_probs_bwd(x, w, t, r, da, dh, workspace=work)
    assert want[0].isfinite().all() and want[1].isfinite().all()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
