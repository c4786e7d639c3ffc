"""One double-pass training step over streamed NF4 layers.

A stack of gated MLP blocks with norms before and after each, a gate and a
residual scale.  The first pass keeps an 8-bit checkpoint of the residual at
every layer boundary; the loss head gives the gradient without keeping logits;
the second pass streams the layers in reverse, recomputes each from its
checkpoint and runs its backward (doublepass/src/backward.rs:419-524).

    python -m examples.double_pass_step [--tokens 2048 --layers 4 --steps 3]
"""
from __future__ import annotations

import argparse
import time
from dataclasses import dataclass
from typing import List

import torch

from aethelstream_amd import checkpoint, gemm, loss, nf4, norm, stream

ALPHA = 0.5  # residual scale of every block


@dataclass
class Model:
    """Layers' NF4 matrices in pinned host memory, small vectors and the head on
    the device."""

    layout: stream.LayerLayout
    pinned: List[stream.PinnedBuffer]
    dbuf: stream.VramDoubleBuffer
    w_pre: List[torch.Tensor]   # one for each layer, then the final norm's
    w_post: List[torch.Tensor]
    gate: List[torch.Tensor]
    head: torch.Tensor          # bf16 [V, d]


def build(layers: int, d: int, ff: int, vocab: int, seed: int = 0):
    """A random model, and its layers' weights as Nf4Weight for a check."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    layout = stream.LayerLayout([("gate", ff, d), ("up", ff, d), ("down", d, ff)])
    pinned, weights = [], []
    for _ in range(layers):
        ws = [nf4.quantize_weight(randn(r, c) * c ** -0.5, double_quant=True)
              for r, c in ((ff, d), (ff, d), (d, ff))]
        buf = stream.PinnedBuffer(layout.nbytes)
        layout.pack_into(buf.tensor, ws)
        pinned.append(buf)
        weights.append(ws)
    model = Model(layout, pinned, stream.VramDoubleBuffer(layout.nbytes),
                  [1 + 0.1 * randn(d) for _ in range(layers + 1)],
                  [1 + 0.1 * randn(d) for _ in range(layers)],
                  [1 + 0.2 * randn(d) for _ in range(layers)],
                  (randn(vocab, d) * 1.5 * d ** -0.5).to(torch.bfloat16))
    return model, weights


def step(model: Model, x: torch.Tensor, targets: torch.Tensor) -> dict:
    """Losses and every gradient for embeddings x (fp32 [M, d])."""
    layers = len(model.pinned)
    current = torch.cuda.current_stream()
    kept = []  # checkpoints of the residual that each layer starts from

    # First pass: one residual, overwritten at every boundary.
    res = x.clone()
    y, rms = norm.rms_norm_fwd(res, model.w_pre[0])
    state = {"y": y, "rms": rms}

    def forward(l, w):
        kept.append(checkpoint.encode(res))
        hidden = gemm.linear_swiglu(state["y"], w[0], w[1])
        h = gemm.linear_fwd(hidden, w[2])
        b = norm.block_norm_fwd(h, res, model.w_pre[l + 1], model.w_post[l], model.gate[l], ALPHA,
                                out=res)
        state["y"], state["rms"] = b.y, b.rms_pre

    stream.run_stack(model.pinned, model.layout, model.dbuf, forward, current)

    # The loss head: gradient of the mean over the tokens that count.
    y = state["y"]
    losses, lse = loss.linear_cross_entropy(y, model.head, targets)
    count = (targets != loss.IGNORE_INDEX).sum().clamp(min=1)
    dloss = (1.0 / count).expand(x.shape[0]).float().contiguous()
    dy, dhead = loss.linear_cross_entropy_bwd(y, model.head, targets, lse, dloss)
    grads = {"head": dhead, "w_pre": [None] * (layers + 1), "w_post": [None] * layers,
             "gate": [None] * layers, "layers": [None] * layers}
    # Second pass, in reverse: recompute from the checkpoint, then backward.  Every
    # norm's backward gets the rms of the values it gets: of the last residual,
    # which is still there, then of the checkpoints as they read back, and of the
    # recomputed h.
    state = {"dy": dy, "dres": None, "res": res, "rms": state["rms"]}

    def backward(i, w):
        l = layers - 1 - i
        _, y, rms = checkpoint.decode_norm(kept[l], model.w_pre[l], want_x=False)
        g, u = (t.float() for t in gemm.linear_fwd_grouped(y, w[:2]))
        s = torch.sigmoid(g)
        hidden = (g * s * u).to(torch.bfloat16)
        h = gemm.linear_fwd(hidden, w[2])
        rms_post = (h.float().square().mean(1) + norm.EPS).sqrt()
        b = norm.block_norm_bwd(state["dy"], state["dres"], state["res"], state["rms"],
                                model.w_pre[l + 1], h=h, rms_post=rms_post,
                                w_post=model.w_post[l], gate=model.gate[l], alpha=ALPHA,
                                out=state["dres"])
        dhidden = gemm.linear_dgrad(b.dh, w[2]).float()
        dg = (dhidden * u * s * (1 + g * (1 - s))).to(torch.bfloat16)
        du = (dhidden * g * s).to(torch.bfloat16)
        grads["layers"][l] = [*gemm.linear_wgrad_grouped([dg, du], y),
                              gemm.linear_wgrad(b.dh, hidden)]
        grads["w_pre"][l + 1], grads["w_post"][l], grads["gate"][l] = b.dw_pre, b.dw_post, b.dgate
        state["dy"], state["dres"] = gemm.linear_dgrad_sum([dg, du], w[:2]), b.dres
        state["res"], state["rms"] = kept[l], rms

    stream.run_stack(model.pinned[::-1], model.layout, model.dbuf, backward, current)
    b = norm.block_norm_bwd(state["dy"], state["dres"], state["res"], state["rms"],
                            model.w_pre[0])
    grads["w_pre"][0], grads["x"] = b.dw_pre, b.dres
    return {"losses": losses, "loss": losses.sum() / count, "grads": grads}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--d", type=int, default=4096)
    ap.add_argument("--ff", type=int, default=11008)
    ap.add_argument("--vocab", type=int, default=32000)
    ap.add_argument("--steps", type=int, default=3)
    a = ap.parse_args()
    model, _ = build(a.layers, a.d, a.ff, a.vocab)
    x = torch.randn(a.tokens, a.d, device="cuda")
    targets = torch.randint(0, a.vocab, (a.tokens,), device="cuda")
    step(model, x, targets)
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(a.steps):
        out = step(model, x, targets)
    torch.cuda.synchronize()
    ms = (time.perf_counter() - began) / a.steps * 1e3
    print(f"loss {float(out['loss']):.4f}, {ms:.1f} ms a step, "
          f"{a.tokens / ms * 1e3:.0f} tokens/s over {a.layers} layers")


if __name__ == "__main__":
    main()
