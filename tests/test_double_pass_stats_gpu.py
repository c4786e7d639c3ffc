"""The example's second pass hands every norm backward the statistics of the
tensors that it hands it: rms_pre of what ``res`` stands for (the checkpoint's
values where it is one), rms_post of ``h``.

Tolerance: an rms of fp32 values is a sum of d squares, a mean and a root, each
fp32 operation off by U = 2^-24 of its result: 64 U, as for the norms themselves
(a sum of at most 32 terms a thread, then of pairs).  Torch's own sums are taken
in 64 bits."""
import pytest
import torch

from aethelstream_amd import checkpoint, norm
from examples import double_pass_step as dp

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _rms(t):
    return (t.double().square().mean(1) + norm.EPS).sqrt()


@pytest.mark.parametrize("tokens", [1, 77, 300])
def test_statistics_belong_to_their_tensors(monkeypatch, tokens):
    layers = 3
    model, _ = dp.build(layers=layers, d=512, ff=1024, vocab=1001, seed=5)
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(tokens, 512, device="cuda", generator=g)
    targets = torch.randint(0, 1001, (tokens,), device="cuda", generator=g)
    calls = []
    real = norm.block_norm_bwd

    def watched(dy, dres, res, rms_pre, w_pre, h=None, rms_post=None, **kw):
        values = checkpoint.decode(res) if isinstance(res, checkpoint.Checkpoint8) else res
        calls.append((rms_pre, _rms(values), rms_post, None if h is None else _rms(h)))
        return real(dy, dres, res, rms_pre, w_pre, h=h, rms_post=rms_post, **kw)

    monkeypatch.setattr(dp.norm, "block_norm_bwd", watched)
    dp.step(model, x, targets)
    assert len(calls) == layers + 1
    for rms_pre, want, rms_post, want_post in calls:
        assert ((rms_pre.double() - want).abs() <= 64 * U * want).all()
        if want_post is not None:
            assert ((rms_post.double() - want_post).abs() <= 64 * U * want_post).all()
