"""The example's double-pass step (norms around the blocks, 8-bit checkpoints, loss
head, streamed NF4 GEMMs) against autograd of the same model in fp32.

Tolerance: along the chain every activation and gradient is rounded to bf16
(relative rms 2^-8 / sqrt(3) = 0.0023 each, about 8 of them a layer) and the
recompute starts from values with the checkpoint's rounding (a step is about
2.7 / 127 of the rms, rms error 0.6 %, twice a layer).  Over two layers their
root sum of squares is below 0.02; 0.05 leaves room for what a norm or the
softmax amplifies."""
import pytest
import torch

from aethelstream_amd import loss, nf4, norm
from examples import double_pass_step as dp

pytestmark = pytest.mark.gpu


def _reference(model, weights, x, targets):
    def leaf(t):
        return t.detach().float().clone().requires_grad_()

    x = leaf(x)
    w_pre, w_post, gate = ([leaf(t) for t in ts] for ts in (model.w_pre, model.w_post, model.gate))
    layers = [[leaf(nf4.dequant(w)) for w in ws] for ws in weights]
    head = leaf(model.head)

    def normed(v, w):
        return v / (v.square().mean(1, keepdim=True) + norm.EPS).sqrt() * w

    res, y = x, normed(x, w_pre[0])
    for l, (g, u, down) in enumerate(layers):
        h = (torch.nn.functional.silu(y @ g.t()) * (y @ u.t())) @ down.t()
        res = res + dp.ALPHA * gate[l] * normed(h, w_post[l])
        y = normed(res, w_pre[l + 1])
    losses = torch.nn.functional.cross_entropy(y @ head.t(), targets, reduction="none",
                                               ignore_index=loss.IGNORE_INDEX)
    count = (targets != loss.IGNORE_INDEX).sum()
    (losses.sum() / count).backward()
    return losses, x, w_pre, w_post, gate, layers, head


def _off(got, want):
    return float((got.float() - want).norm() / want.norm())


@pytest.mark.parametrize("tokens", [1, 100, 333])
def test_step_matches_autograd(tokens):
    model, weights = dp.build(layers=2, d=512, ff=1024, vocab=3001, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(tokens, 512, device="cuda", generator=g)
    targets = torch.randint(0, 3001, (tokens,), device="cuda", generator=g)
    if tokens > 1:
        targets[tokens // 2] = loss.IGNORE_INDEX
    out = dp.step(model, x, targets)
    losses, rx, w_pre, w_post, gate, layers, head = _reference(model, weights, x, targets)
    assert _off(out["losses"], losses.detach()) < 0.01
    grads = out["grads"]
    assert _off(grads["x"], rx.grad) < 0.05
    assert _off(grads["head"], head.grad) < 0.05
    for got, want in ((grads["w_pre"], w_pre), (grads["w_post"], w_post), (grads["gate"], gate)):
        for a, b in zip(got, want):
            assert _off(a, b.grad) < 0.05
    for got, want in zip(grads["layers"], layers):
        for a, b in zip(got, want):
            assert _off(a, b.grad) < 0.05
