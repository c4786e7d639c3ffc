"""Operators of a double-pass training step beside the streamed GEMMs.

Three families, each through the package's public entry points:

* the loss head: cross entropy of x . W^T without keeping the logits, and its
  gradients (``loss.linear_cross_entropy``, ``loss.linear_cross_entropy_bwd``);
* the norms around a block, with its gate and residual scale, forward and
  backward (``norm.block_norm_fwd``, ``norm.block_norm_bwd``);
* activation checkpoints in 8 bits and their use in the backward pass
  (``checkpoint.encode``, ``decode``, ``decode_norm``, and
  ``norm.block_norm_bwd`` reading one).

The plain forms below are elementary torch operations in 32 bits, rounded once
at the end; ``exact`` states the same definitions in 64 bits.
"""
import math

import torch

own = False

BLOCK = 128                 # checkpoint elements per scale, along a row
SMALLEST = 2.0 ** -126      # of a checkpoint scale: the smallest normal fp32
EPS = 1e-6
IGNORE = -100
ALPHA = 0.7                 # residual scale


# --------------------------------------------------------------------------
# The cases
# --------------------------------------------------------------------------

def listed():
    return [
        # Scoring the last token of a prompt: all latency and weight bytes.
        {"name": "ce_score_one", "op": "ce", "train": False, "m": 1, "v": 32000, "d": 4096},
        # Evaluation of a ragged batch with a vocabulary of odd size.
        {"name": "ce_eval_ragged", "op": "ce", "train": False, "m": 1000, "v": 50021, "d": 5120},
        # Loss and gradients of a short micro-batch.
        {"name": "ce_train_short", "op": "ce", "train": True, "m": 77, "v": 32000, "d": 4096},
        # Loss and gradients of a full micro-batch, large vocabulary: the
        # largest case.
        {"name": "ce_train_full", "op": "ce", "train": True, "m": 4096, "v": 128000, "d": 8192},
        # The norms at a layer boundary for one new token: the smallest call.
        {"name": "norm_fwd_one", "op": "norm_fwd", "m": 1, "d": 4096, "post": True, "gate": False},
        # ... of a training micro-batch of a 70B-sized layer.
        {"name": "norm_fwd_full", "op": "norm_fwd", "m": 8192, "d": 8192, "post": True,
         "gate": True},
        # Their backward pass at a ragged micro-batch without a norm after the
        # block, and a full one with every part.
        {"name": "norm_bwd_ragged", "op": "norm_bwd", "m": 1000, "d": 5120, "post": False,
         "gate": True, "bits8": False},
        {"name": "norm_bwd_full", "op": "norm_bwd", "m": 8192, "d": 8192, "post": True,
         "gate": True, "bits8": False},
        # The same backward reading the residual from its 8-bit checkpoint.
        {"name": "norm_bwd_bits8", "op": "norm_bwd", "m": 4096, "d": 4096, "post": True,
         "gate": False, "bits8": True},
        # A block's residual checkpointed and read back (fp32), and a wide
        # bf16 activation whose rows end inside a block.
        {"name": "ckpt_residual", "op": "ckpt", "m": 8192, "d": 8192, "bf16": False},
        {"name": "ckpt_hidden", "op": "ckpt", "m": 777, "d": 13820, "bf16": True},
        # The recompute's first step: checkpoint to residual and normed input.
        {"name": "ckpt_recompute", "op": "recompute", "m": 4096, "d": 8192},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _multiple(rng, lo, hi, step):
    return max(lo, _log_int(rng, lo, hi) // step * step)


def draw(rng):
    """A case of the ranges that the listed ones stand for: 1 to 8192 tokens,
    any vocabulary, rows of any width that the formats allow."""
    biggest = max(work(c)["flops"] for c in listed())
    most = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(("ce", "ce", "norm_fwd", "norm_bwd", "norm_bwd", "ckpt", "recompute"))
        if op == "ce":
            case = {"op": op, "train": rng.random() < 0.6, "m": _log_int(rng, 1, 8192),
                    "v": _log_int(rng, 1000, 128000), "d": _multiple(rng, 1024, 8192, 8)}
        else:
            case = {"op": op, "m": _log_int(rng, 1, 8192), "d": _multiple(rng, 512, 16384, 4)}
            if op in ("norm_fwd", "norm_bwd"):
                case.update(post=rng.random() < 0.6, gate=rng.random() < 0.5)
            if op == "norm_bwd":
                case["bits8"] = rng.random() < 0.5
            if op == "ckpt":
                case["bf16"] = rng.random() < 0.5
        w = work(case)
        if w["flops"] <= biggest and w["bytes"] <= most:
            return case


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------

def _normal(shape, seed, sigma=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * sigma).to(dtype)


def _residual(m, d, seed):
    """A residual stream: normal values, a few channels far larger."""
    x = _normal((m, d), seed, 1.5)
    loud = _normal((d,), seed + 1)
    return x * torch.where(loud > 2.5, 12.0, 1.0)


def _coded(x):
    """Codes and scales of an 8-bit checkpoint of x, in plain torch."""
    m, d = x.shape
    blocks = (d + BLOCK - 1) // BLOCK
    pad = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - d)).view(m, blocks, BLOCK)
    scale = (pad.abs().amax(2) / 127.0).clamp(min=SMALLEST)
    q = torch.round(pad * (1.0 / scale)[:, :, None])
    return q.view(m, -1)[:, :d].to(torch.int8).contiguous(), scale


def _values(codes, scales):
    """What 8-bit codes stand for, in the scales' type."""
    m, d = codes.shape
    return codes.to(scales.dtype) * scales.repeat_interleave(BLOCK, 1)[:, :d]


def prepare(case, seed):
    op, m, d = case["op"], case["m"], case["d"]
    seed = seed * 1000
    s = {"op": op}
    if op == "ce":
        v = case["v"]
        g = torch.Generator(device="cuda").manual_seed(seed)
        s["train"] = case["train"]
        s["x"] = _normal((m, d), seed + 1, 1.0, torch.bfloat16)
        s["w"] = _normal((v, d), seed + 2, 0.02, torch.bfloat16)
        t = torch.randint(0, v, (m,), device="cuda", generator=g)
        skip = torch.rand((m,), device="cuda", generator=g) < 0.1
        s["targets"] = torch.where(skip & (torch.arange(m, device="cuda") > 0), IGNORE, t)
        s["dloss"] = torch.full((m,), 1.0 / m, device="cuda")
        return s
    if op == "ckpt":
        s["x"] = _residual(m, d, seed).to(torch.bfloat16 if case["bf16"] else torch.float32)
        return s
    res = _residual(m, d, seed)
    s["w_pre"] = 1.0 + _normal((d,), seed + 3, 0.1)
    if op == "recompute":
        s["codes"], s["scales"] = _coded(res)
        return s
    s["h"] = _normal((m, d), seed + 4, 0.5, torch.bfloat16)
    s["w_post"] = 1.0 + _normal((d,), seed + 5, 0.1) if case["post"] else None
    s["gate"] = _normal((d,), seed + 6, 0.5) if case["gate"] else None
    if op == "norm_fwd":
        s["res"] = res
        return s
    s["bits8"] = case["bits8"]
    if case["bits8"]:
        s["codes"], s["scales"] = _coded(res)
        res = _values(s["codes"], s["scales"])
    else:
        s["res"] = res
    s["rms_pre"] = (res.square().mean(1) + EPS).sqrt()
    s["rms_post"] = (s["h"].float().square().mean(1) + EPS).sqrt() if case["post"] else None
    s["dy"] = _normal((m, d), seed + 7, 1e-3, torch.bfloat16)
    s["dres"] = _normal((m, d), seed + 8, 1e-3)
    return s


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from aethelstream_amd import checkpoint, loss, norm
    op = s["op"]
    if op == "ce":
        out, lse = loss.linear_cross_entropy(s["x"], s["w"], s["targets"], ignore_index=IGNORE)
        if not s["train"]:
            return {"loss": out, "lse": lse}
        dx, dw = loss.linear_cross_entropy_bwd(s["x"], s["w"], s["targets"], lse, s["dloss"],
                                               ignore_index=IGNORE)
        return {"loss": out, "lse": lse, "dx": dx, "dw": dw}
    if op == "norm_fwd":
        r = norm.block_norm_fwd(s["h"], s["res"], s["w_pre"], w_post=s["w_post"], gate=s["gate"],
                                alpha=ALPHA, eps=EPS)
        return _some(res=r.res, y=r.y, rms_pre=r.rms_pre, rms_post=r.rms_post)
    if op == "norm_bwd":
        res = checkpoint.Checkpoint8(s["codes"], s["scales"]) if s["bits8"] else s["res"]
        r = norm.block_norm_bwd(s["dy"], s["dres"], res, s["rms_pre"], s["w_pre"], h=s["h"],
                                rms_post=s["rms_post"], w_post=s["w_post"], gate=s["gate"],
                                alpha=ALPHA)
        return _some(dres=r.dres, dh=r.dh, dw_pre=r.dw_pre, dw_post=r.dw_post, dgate=r.dgate)
    if op == "ckpt":
        c = checkpoint.encode(s["x"])
        return {"scales": c.scales, "x": checkpoint.decode(c, dtype=s["x"].dtype)}
    c = checkpoint.Checkpoint8(s["codes"], s["scales"])
    x, y, rms = checkpoint.decode_norm(c, s["w_pre"], eps=EPS)
    return {"x": x, "y": y, "rms": rms}


def _some(**outs):
    return {k: v for k, v in outs.items() if v is not None}


def _plain(s):
    op = s["op"]
    if op == "ce":
        return _plain_ce(s)
    if op == "norm_fwd":
        h = s["h"].float()
        rms_post = None
        if s["w_post"] is not None:
            rms_post = (h.square().mean(1) + EPS).sqrt()
            h = h / rms_post[:, None] * s["w_post"]
        if s["gate"] is not None:
            h = h * s["gate"]
        res = s["res"] + ALPHA * h
        rms = (res.square().mean(1) + EPS).sqrt()
        y = (res / rms[:, None] * s["w_pre"]).to(torch.bfloat16)
        return _some(res=res, y=y, rms_pre=rms, rms_post=rms_post)
    if op == "norm_bwd":
        return _plain_norm_bwd(s)
    if op == "ckpt":
        codes, scales = _coded(s["x"])
        return {"scales": scales, "x": _values(codes, scales).to(s["x"].dtype)}
    x = _values(s["codes"], s["scales"])
    rms = (x.square().mean(1) + EPS).sqrt()
    return {"x": x, "y": (x / rms[:, None] * s["w_pre"]).to(torch.bfloat16), "rms": rms}


def _plain_ce(s):
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    top = z.amax(1)
    z -= top[:, None]
    kept = s["targets"] != IGNORE
    at = s["targets"].clamp(min=0)
    hit = z.gather(1, at[:, None])[:, 0]
    z = z.exp_()
    total = z.sum(1)
    out = torch.where(kept, total.log() - hit, 0.0)
    lse = total.log() + top
    if not s["train"]:
        return {"loss": out, "lse": lse}
    g = z.mul_((1.0 / total)[:, None])
    rows = torch.arange(g.shape[0], device=g.device)
    g[rows, at] -= 1.0
    g *= torch.where(kept, s["dloss"], 0.0)[:, None]
    return {"loss": out, "lse": lse, "dx": (g @ w).to(torch.bfloat16),
            "dw": (g.t() @ x).to(torch.bfloat16)}


def _plain_norm_bwd(s):
    res = _values(s["codes"], s["scales"]) if s["bits8"] else s["res"]
    hat = res / s["rms_pre"][:, None]
    dy = s["dy"].float()
    e = dy * s["w_pre"]
    g = s["dres"] + (e - hat * (e * hat).mean(1, keepdim=True)) / s["rms_pre"][:, None]
    dw_pre = (dy * hat).sum(0)
    h = s["h"].float()
    if s["w_post"] is not None:
        h = h / s["rms_post"][:, None]
    along = ALPHA * (g * h).sum(0)
    e = ALPHA * g
    dgate = dw_post = None
    if s["gate"] is not None:
        dgate = along * s["w_post"] if s["w_post"] is not None else along
        e = e * s["gate"]
    if s["w_post"] is not None:
        dw_post = along * s["gate"] if s["gate"] is not None else along
        e = e * s["w_post"]
        e = (e - h * (e * h).mean(1, keepdim=True)) / s["rms_post"][:, None]
    return _some(dres=g, dh=e.to(torch.bfloat16), dw_pre=dw_pre, dw_post=dw_post, dgate=dgate)


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    op, m, d = case["op"], case["m"], case["d"]
    if op == "ce":
        v = case["v"]
        # x, W and targets in, loss and lse out; the logits are products of
        # length d.  A training pass reads dloss and writes dx and dW too, and
        # multiplies four times: logits, logits again (they are not kept), dx
        # and dW.
        moved = 2 * (m + v) * d + 16 * m
        if not case["train"]:
            return {"bytes": moved, "flops": 2 * m * v * d}
        return {"bytes": moved + 2 * (m + v) * d + 4 * m, "flops": 8 * m * v * d}
    n = m * d
    scales = 4 * m * ((d + BLOCK - 1) // BLOCK)
    vectors = 4 * d * (1 + case.get("post", 0) + case.get("gate", 0))
    rows = 4 * m * (1 + case.get("post", 0))
    if op == "norm_fwd":      # h, res in; res, y out
        return {"bytes": 12 * n + vectors + rows, "flops": 12 * n}
    if op == "norm_bwd":      # dy, dres, res or its codes, h in; dres, dh out
        res = n + scales if case["bits8"] else 4 * n
        return {"bytes": 14 * n + res + 2 * vectors + rows, "flops": 24 * n}
    if op == "ckpt":          # x in, codes and scales out and in again, x out
        size = 2 if case["bf16"] else 4
        return {"bytes": 2 * (size + 1) * n + 2 * scales, "flops": 4 * n}
    return {"bytes": (1 + 4 + 2) * n + scales + 4 * d + 4 * m, "flops": 6 * n}


# --------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "ce":
        return _exact_ce(s)
    if op == "ckpt":
        x = s["x"].double()
        m, d = x.shape
        blocks = (d + BLOCK - 1) // BLOCK
        padded = torch.zeros(m, blocks * BLOCK, dtype=torch.float64, device=x.device)
        padded[:, :d] = x
        parts = padded.view(m, blocks, BLOCK)
        scales = torch.clamp(parts.abs().max(dim=2).values / 127, min=SMALLEST)
        back = torch.round(parts / scales.unsqueeze(2)) * scales.unsqueeze(2)
        return {"scales": scales, "x": back.reshape(m, -1)[:, :d]}

    def normed(t):
        rms = torch.sqrt((t * t).sum(1) / t.shape[1] + EPS)
        return t / rms.unsqueeze(1), rms

    w_pre = s["w_pre"].double()
    if op == "recompute":
        x = _values(s["codes"], s["scales"].double())
        hat, rms = normed(x)
        return {"x": x, "y": hat * w_pre, "rms": rms}
    h = s["h"].double()
    one = torch.ones_like(w_pre)
    gate = one if s["gate"] is None else s["gate"].double()
    w_post = one if s["w_post"] is None else s["w_post"].double()
    if op == "norm_fwd":
        hat, rms_post = normed(h) if s["w_post"] is not None else (h, None)
        res = s["res"].double() + ALPHA * gate * w_post * hat
        y, rms = normed(res)
        return _some(res=res, y=y * w_pre, rms_pre=rms, rms_post=rms_post)
    # The row's rms values are inputs of the backward pass.
    d = h.shape[1]
    res = _values(s["codes"], s["scales"].double()) if s["bits8"] else s["res"].double()
    rms = s["rms_pre"].double().unsqueeze(1)
    hat = res / rms
    dy = s["dy"].double()
    dhat = dy * w_pre
    g = s["dres"].double() + (dhat - hat * ((dhat * hat).sum(1, keepdim=True) / d)) / rms
    du = ALPHA * gate * g
    if s["w_post"] is None:
        return _some(dres=g, dh=du, dw_pre=(dy * hat).sum(0),
                     dgate=None if s["gate"] is None else (ALPHA * g * h).sum(0))
    rms_post = s["rms_post"].double().unsqueeze(1)
    hhat = h / rms_post
    dhat = du * w_post
    dh = (dhat - hhat * ((dhat * hhat).sum(1, keepdim=True) / d)) / rms_post
    return _some(dres=g, dh=dh, dw_pre=(dy * hat).sum(0), dw_post=(du * hhat).sum(0),
                 dgate=None if s["gate"] is None else (ALPHA * g * hhat * w_post).sum(0))


def _exact_ce(s):
    x, w, t = s["x"].double(), s["w"].double(), s["targets"]
    z = torch.matmul(x, w.t())
    lse = torch.logsumexp(z, 1)
    kept = t != IGNORE
    at = torch.where(kept, t, 0).unsqueeze(1)
    loss = torch.where(kept, lse - torch.gather(z, 1, at).squeeze(1), torch.zeros_like(lse))
    if not s["train"]:
        return {"loss": loss, "lse": lse}
    z = torch.exp(z - lse.unsqueeze(1))
    z.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    z = z * torch.where(kept, s["dloss"].double(), torch.zeros_like(lse)).unsqueeze(1)
    return {"loss": loss, "lse": lse, "dx": torch.matmul(z, w), "dw": torch.matmul(z.t(), x)}
