"""Kept logits of the log probabilities: they belong to one shape, and the gradients take
them piece by piece of the vocabulary."""
import pytest
import torch

import test_linear_ce_gpu as ce
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
