"""Log probabilities and their gradients over columns behind whole rounds of large tiles,
and in the smallest tiles for few tokens, against 64 bits (tolerances:
test_linear_logprob_gpu.py).  test_linear_logprob_plan.py shows that the shapes are cut
so."""
import pytest
import torch

import test_linear_ce_gpu as ce
import test_linear_logprob_gpu as lp
import test_linear_logprob_plan as plan
from aethelstream_amd import loss

pytestmark = pytest.mark.gpu


def _gradients(m, v, d):
    """Forward, kept logits and logits made again, and the gradients of both."""
    x, w, t, da = ce._inputs(m, v, d, seed=m + v)
    # Targets among the last columns too, and on both sides of the launches' border.
    t[::3] = v - 1 - torch.arange(len(t[::3]), device="cuda") % min(v, 70)
    dh = ce._randn((m,), 9, 0.5, torch.float32)
    r = loss.linear_log_probs(x, w, t, keep_logits=True)
    s = loss.linear_log_probs(x, w, t, keep_logits=False)
    lp._check_forward(x, w, t, r)
    for name in ("logp", "entropy", "lse"):
        assert torch.equal(getattr(r, name), getattr(s, name))
    got, want = (loss.linear_log_probs_bwd(x, w, t, o, da, dh) for o in (r, s))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    lp._check_backward(x, w, t, da, dh, r, *got)
    return x, w, t


@pytest.mark.parametrize("m,v,d,first,width", plan.SPLITS)
def test_two_launches(m, v, d, first, width):
    print(m, v, d, flush=True)
    assert plan.in_two_launches(m, v, d, first, width)
    x, w, t = _gradients(m, v, d)
    lp._check_forward(x, w, t, loss.linear_log_probs(x, w, t, top_k=9))


@pytest.mark.parametrize("m,v,d,first,width", plan.SPLITS[:6])
def test_ranks_over_two_launches(m, v, d, first, width):
    """Equal logits on both sides of the border, and all of them equal."""
    print(m, v, d, flush=True)
    x, w = lp._grid(m, v, d, seed=m, levels=1)
    w[first:] = w[:v - first]
    t = torch.zeros(m, dtype=torch.int64, device="cuda")
    for k in (1, 20):
        lp._check_ranks(x, w, loss.linear_log_probs(x, w, t, top_k=k), k)
    x[:] = 0
    lp._check_ranks(x, w, loss.linear_log_probs(x, w, t, top_k=32), 32)


@pytest.mark.parametrize("m,v,d", plan.FEW + plan.NEXT_TO_FEW)
def test_few_tokens(m, v, d):
    print(m, v, d, flush=True)
    x, w, t = _gradients(m, v, d)
    for k in (1, 8, 32):
        lp._check_forward(x, w, t, loss.linear_log_probs(x, w, t, top_k=k))


@pytest.mark.parametrize("m,v,d", plan.FEW + plan.NEXT_TO_FEW)
@pytest.mark.parametrize("levels", [1, 8])
def test_ranks_of_few_tokens(m, v, d, levels):
    print(m, v, d, flush=True)
    x, w = lp._grid(m, v, d, seed=v + m, levels=levels)
    if levels == 1:
        w[v // 2:] = w[:v - v // 2]  # every logit twice at least
    t = torch.zeros(m, dtype=torch.int64, device="cuda")
    for k in (1, 8, 32):
        lp._check_ranks(x, w, loss.linear_log_probs(x, w, t, top_k=k), k)
    x[:m // 2 + 1] = 0
    lp._check_ranks(x, w, loss.linear_log_probs(x, w, t, top_k=32), 32)
