"""One policy-training step of a small attention model over NF4 weights.

Queries and keys get their heads' norms and the rotation by position between their
products and attention; the loss is the advantage-weighted log probability of the
given tokens with an entropy bonus, taken from the hidden states and the head (which
keeps the logits for the gradients while they take no more memory than itself); an
AdamW step updates the fp32 masters, the norms' weights and the bf16 head, and the
masters are quantized again.  (The attention between is plain torch in fp32.)

    python -m examples.policy_step [--tokens 512 --steps 20]
"""
from __future__ import annotations

import argparse
import time
from dataclasses import dataclass
from typing import List

import torch

from aethelstream_amd import gemm, loss, nf4, norm, optim, rotary

BONUS = 0.01  # of the entropy
LR, BETAS, DECAY = 1e-3, (0.9, 0.95), 0.1


@dataclass
class Model:
    """q, k, v and output projections in NF4 with fp32 masters, the norms' weights
    (before the block, after it, of query and key heads), and the bf16 head."""

    heads: int
    kv_heads: int
    weights: List[nf4.Nf4Weight]
    masters: List[torch.Tensor]
    norms: List[torch.Tensor]
    head: torch.Tensor
    rope: rotary.Rotary
    state: optim.AdamWState

    def params(self) -> List[torch.Tensor]:
        return [*self.masters, *self.norms, self.head]


def build(d: int, heads: int, kv_heads: int, head_size: int, vocab: int, bits: int = 8,
          seed: int = 0) -> Model:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    rows = [heads * head_size, kv_heads * head_size, kv_heads * head_size, d]
    masters = [randn(r, c) * c ** -0.5 for r, c in zip(rows, (d, d, d, heads * head_size))]
    weights = [nf4.quantize_weight(w, double_quant=True) for w in masters]
    norms = [1 + 0.1 * randn(n) for n in (d, d, head_size, head_size)]
    head = (randn(vocab, d) * 1.5 * d ** -0.5).to(torch.bfloat16)
    f, scale = rotary.frequencies(head_size)
    rope = rotary.Rotary.from_frequencies(f, scale=scale)
    return Model(heads, kv_heads, weights, masters, norms, head, rope,
                 optim.adamw_state([*masters, *norms, head], bits))


def _attention(q, k, v):
    """Causal attention of [M, heads, size], in fp32: the output, and what its
    gradients need."""
    m, h, size = q.shape
    share = h // k.shape[1]
    q = q.float().transpose(0, 1)
    k, v = (t.float().repeat_interleave(share, 1).transpose(0, 1) for t in (k, v))
    s = torch.matmul(q, k.transpose(1, 2).contiguous()) * size ** -0.5
    late = torch.ones(m, m, dtype=torch.bool, device=q.device).triu(1)
    p = torch.softmax(s.masked_fill(late, float("-inf")), 2)
    return torch.matmul(p, v).transpose(0, 1).to(torch.bfloat16).contiguous(), (q, k, v, p)


def _attention_bwd(do, saved, kv_heads):
    q, k, v, p = saved
    do = do.float().transpose(0, 1)
    dv = torch.matmul(p.transpose(1, 2).contiguous(), do)
    dp = torch.matmul(do, v.transpose(1, 2).contiguous())
    ds = p * (dp - (dp * p).sum(2, keepdim=True)) * q.shape[2] ** -0.5
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(1, 2).contiguous(), q)

    def back(t, heads):  # the heads that share one, summed
        t = t.transpose(0, 1)
        return t.reshape(t.shape[0], heads, -1, t.shape[2]).sum(2).to(torch.bfloat16).contiguous()

    return back(dq, q.shape[0]), back(dk, kv_heads), back(dv, kv_heads)


def step(model: Model, x: torch.Tensor, positions: torch.Tensor, targets: torch.Tensor,
         advantages: torch.Tensor) -> dict:
    """Loss, its parts and every gradient for embeddings x (fp32 [M, d])."""
    m = x.shape[0]
    w_in, w_out, w_q, w_k = model.norms
    y, rms = norm.rms_norm_fwd(x, w_in)
    q, k, v = gemm.linear_fwd_grouped(y, model.weights[:3])
    q, k, v = (t.view(m, h, -1) for t, h in ((q, model.heads), (k, model.kv_heads),
                                            (v, model.kv_heads)))
    qr, kr = rotary.apply(q, k, positions, model.rope, w_q, w_k)
    o, saved = _attention(qr, kr, v)
    h = gemm.linear_fwd(o.view(m, -1), model.weights[3])
    b = norm.block_norm_fwd(h, x, w_out)
    out = loss.linear_log_probs(b.y, model.head, targets)
    # Minus the mean over all tokens of advantage * log probability + bonus * entropy.
    value = -(advantages * out.logp + BONUS * out.entropy).mean()
    dlogp = -advantages / m
    dentropy = torch.full_like(dlogp, -BONUS / m)

    dy, dhead = loss.linear_log_probs_bwd(b.y, model.head, targets, out, dlogp, dentropy)
    n = norm.block_norm_bwd(dy, None, b.res, b.rms_pre, w_out, h=h)
    do = gemm.linear_dgrad(n.dh, model.weights[3])
    dq, dk, dv = _attention_bwd(do.view(m, model.heads, -1), saved, model.kv_heads)
    r = rotary.apply_bwd(dq, dk, positions, model.rope, q=q, k=k, w_q=w_q, w_k=w_k, out_q=dq,
                         out_k=dk)
    dqkv = [t.view(m, -1) for t in (r.dq, r.dk, dv)]
    dx = gemm.linear_dgrad_sum(dqkv, model.weights[:3])
    first = norm.block_norm_bwd(dx, n.dres, x, rms, w_in)
    matrices = [*gemm.linear_wgrad_grouped(dqkv, y), gemm.linear_wgrad(n.dh, o.view(m, -1))]
    return {"loss": value, "logp": out.logp, "entropy": out.entropy, "x": first.dres,
            "grads": [*matrices, first.dw_pre, n.dw_pre, r.dw_q, r.dw_k, dhead]}


def update(model: Model, grads: List[torch.Tensor], t: int) -> None:
    """Step t (from 1 on) of every parameter, and the masters in NF4 again."""
    norms = torch.stack([g.float().norm() for g in grads])
    clip = (1.0 / (norms.norm() + 1e-6)).clamp(max=1.0).reshape(1)
    optim.adamw_step(model.params(), grads, model.state, t, lr=LR, betas=BETAS,
                     weight_decay=DECAY, grad_scale=clip)
    for w, master in zip(model.weights, model.masters):
        nf4.requantize_(w, master)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--d", type=int, default=2048)
    ap.add_argument("--heads", type=int, default=16)
    ap.add_argument("--kv-heads", type=int, default=4)
    ap.add_argument("--vocab", type=int, default=32000)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    model = build(a.d, a.heads, a.kv_heads, a.d // a.heads, a.vocab)
    x = torch.randn(a.tokens, a.d, device="cuda")
    positions = torch.arange(a.tokens, device="cuda")
    targets = torch.randint(0, a.vocab, (a.tokens,), device="cuda")
    advantages = torch.randn(a.tokens, device="cuda")
    out = step(model, x, positions, targets, advantages)
    torch.cuda.synchronize()
    began = time.perf_counter()
    for t in range(1, a.steps + 1):
        out = step(model, x, positions, targets, advantages)
        update(model, out["grads"], t)
    torch.cuda.synchronize()
    ms = (time.perf_counter() - began) / a.steps * 1e3
    print(f"loss {float(out['loss']):.4f}, entropy {float(out['entropy'].mean()):.3f}, "
          f"{ms:.2f} ms a step of {a.tokens} tokens")


if __name__ == "__main__":
    main()
