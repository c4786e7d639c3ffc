"""The example's policy step (norms and rotation of queries and keys, log
probabilities with an entropy bonus, AdamW with 8-bit moments, NF4 weights quantized
again) against autograd of the same model in fp32, and its update against the
formula.

Tolerance: along the chain every activation and gradient is rounded to bf16
(relative rms 2^-8 / sqrt(3) = 0.0023 each, about 12 of them); their root sum of
squares is below 0.01, and 0.05 leaves room for what norms and softmax amplify."""
import pytest
import torch

from aethelstream_amd import loss, nf4, norm, optim
from examples import policy_step as ps

pytestmark = pytest.mark.gpu


def _reference(model, x, positions, targets, advantages):
    def leaf(t):
        return t.detach().float().clone().requires_grad_()

    x = leaf(x)
    ws = [leaf(nf4.dequant(w)) for w in model.weights]
    w_in, w_out, w_q, w_k = norms = [leaf(t) for t in model.norms]
    head = leaf(model.head)
    m = x.shape[0]

    def normed(v, w):
        return v / (v.square().mean(-1, keepdim=True) + norm.EPS).sqrt() * w

    def turned(t):
        half = t.shape[2] // 2
        f = 10000.0 ** (-torch.arange(half, device=t.device).double() / half)
        a = positions.double()[:, None] * f
        cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
        u, v = t[..., :half], t[..., half:]
        return torch.cat((u * cos - v * sin, v * cos + u * sin), 2)

    y = normed(x, w_in)
    q, k, v = ((y @ w.t()).view(m, h, -1) for w, h in zip(
        ws, (model.heads, model.kv_heads, model.kv_heads)))
    q, k = turned(normed(q, w_q)), turned(normed(k, w_k))
    share = model.heads // model.kv_heads
    k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    s = (q.transpose(0, 1) @ k.permute(1, 2, 0).contiguous()) * q.shape[2] ** -0.5
    late = torch.ones(m, m, dtype=torch.bool, device=x.device).triu(1)
    p = torch.softmax(s.masked_fill(late, float("-inf")), 2)
    o = (p @ v.transpose(0, 1).contiguous()).transpose(0, 1).reshape(m, -1)
    z = normed(x + o @ ws[3].t(), w_out) @ head.t()
    l = torch.log_softmax(z, 1)
    kept = targets != loss.IGNORE_INDEX
    logp = torch.where(kept, l.gather(1, targets.clamp(min=0)[:, None])[:, 0], 0.0)
    entropy = -(l.exp() * l).sum(1)
    value = -(advantages * logp + ps.BONUS * entropy).mean()
    value.backward()
    return value, logp, entropy, x.grad, [t.grad for t in (*ws, *norms, head)]


def _off(got, want):
    return float((got.float() - want).norm() / want.norm())


def _inputs(tokens, d, vocab, seed=4):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, d, device="cuda", generator=g)
    targets = torch.randint(0, vocab, (tokens,), device="cuda", generator=g)
    if tokens > 2:
        targets[tokens // 2] = loss.IGNORE_INDEX
    advantages = torch.randn(tokens, device="cuda", generator=g)
    return x, torch.arange(tokens, device="cuda") + 5, targets, advantages


@pytest.mark.parametrize("tokens", [2, 77, 300])
def test_gradients_match_autograd(tokens):
    model = ps.build(512, 8, 2, 64, 3001, seed=3)
    args = _inputs(tokens, 512, 3001)
    out = ps.step(model, *args)
    value, logp, entropy, dx, grads = _reference(model, *args)
    assert abs(float(out["loss"] - value.detach())) < 0.01 * float(logp.detach().abs().mean())
    assert _off(out["logp"], logp.detach()) < 0.01
    assert _off(out["entropy"], entropy.detach()) < 0.01
    assert _off(out["x"], dx) < 0.05
    for got, want in zip(out["grads"], grads):
        assert got.shape == want.shape and _off(got, want) < 0.05


@pytest.mark.parametrize("bits", [8, 32])
def test_update(bits):
    """Two updates: the masters, vectors and head as the formula has them, and the NF4
    weights the masters' quantization."""
    model = ps.build(256, 4, 4, 64, 1001, bits=bits, seed=5)
    args = _inputs(50, 256, 1001)
    for t in (1, 2):
        grads = ps.step(model, *args)["grads"]
        clip = min(1.0, 1.0 / (float(torch.stack([g.float().norm() for g in grads]).norm())
                               + 1e-6))
        c = optim.coefficients(t, ps.LR, ps.BETAS, 1e-8, ps.DECAY)
        m0, v0 = (a.double() for a in optim.moments(model.state))
        want = []
        for p, g, a in zip(model.params(), grads, model.state.starts()):
            n = p.numel()
            g = g.double().reshape(-1) * clip
            m = m0[a:a + n] * c[0] + g * c[1]
            v = v0[a:a + n] * c[2] + g * g * c[3]
            want.append(p.double().reshape(-1) * c[4] - m / (v.sqrt() * c[6] + c[7]) * c[5])
        ps.update(model, grads, t)
        for p, w in zip(model.params(), want):
            # The update's own errors are 2^-18 of lr at most (a clipping factor of two
            # roundings); a bf16 parameter is rounded.
            step = 2.0 ** -8 if p.dtype == torch.bfloat16 else 2.0 ** -23
            assert ((p.double().reshape(-1) - w).abs() <= step * w.abs() + 2.0 ** -16 * c[5]).all()
        for w, master in zip(model.weights, model.masters):
            again = nf4.quantize_weight(master, double_quant=True)
            assert torch.equal(w.packed, again.packed) and torch.equal(w.absmax_q, again.absmax_q)
