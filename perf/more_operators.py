"""Operators of a training step next to the streamed GEMMs and the loss head.

Three families, each through the package's public entry points:

* queries and keys between their GEMMs and attention: a norm for each head and
  the rotation by position in one pass, or the rotation alone, forward and
  backward (``rotary.apply``, ``rotary.apply_bwd``);
* log probabilities of given tokens under a linear head, their entropy and the
  top alternatives without keeping the logits, and the gradients
  (``loss.linear_log_probs``, ``loss.linear_log_probs_bwd``);
* an AdamW step over many tensors at once with its moments in 32 or 8 bits
  (``optim.adamw_step``, ``optim.moments``).

The plain forms below are elementary torch operations in 32 bits (angles in 64),
rounded once at the end; ``exact`` states the same definitions in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-6                  # of the norms
IGNORE = -100
BLOCK = 128                 # moments in 8 bits that share a scale
SMALLEST = 2.0 ** -126      # of such a scale
OFFSET = 2.0 ** -15         # where the codes' exponents begin
LR, BETAS, ADAM_EPS, DECAY = 3e-4, (0.9, 0.95), 1e-8, 0.1


# --------------------------------------------------------------------------
# The cases
# --------------------------------------------------------------------------

def listed():
    return [
        # One new token of a 7B-sized layer: the smallest call, all latency.
        {"name": "rotary_one", "op": "rotary", "bwd": False, "m": 1, "hq": 32, "hk": 32, "d": 128,
         "rot": 128, "pairs": "half", "norm": True, "far": True, "bf16": True, "fused": False},
        # A training micro-batch of a 70B-sized layer, with norms.
        {"name": "rotary_full", "op": "rotary", "bwd": False, "m": 8192, "hq": 64, "hk": 8,
         "d": 128, "rot": 128, "pairs": "half", "norm": True, "far": False, "bf16": True,
         "fused": False},
        # Adjacent pairs over half of each head, frequencies scaled for a long
        # context, ragged token count, q and k inside one row with v.
        {"name": "rotary_long_ragged", "op": "rotary", "bwd": False, "m": 1000, "hq": 40, "hk": 10,
         "d": 128, "rot": 64, "pairs": "adjacent", "norm": False, "far": True, "bf16": True,
         "fused": True},
        # Gradients of the full micro-batch, norms' weights included.
        {"name": "rotary_bwd_full", "op": "rotary", "bwd": True, "m": 8192, "hq": 64, "hk": 8,
         "d": 128, "rot": 128, "pairs": "half", "norm": True, "far": False, "bf16": True,
         "fused": False},
        # Gradients in fp32 of heads whose size is no power of two.
        {"name": "rotary_bwd_ragged", "op": "rotary", "bwd": True, "m": 777, "hq": 12, "hk": 12,
         "d": 80, "rot": 40, "pairs": "half", "norm": True, "far": False, "bf16": False,
         "fused": False},
        # The next token's most likely alternatives after a prompt.
        {"name": "logprob_one", "op": "logprob", "train": False, "m": 1, "v": 32000, "d": 4096,
         "k": 8},
        # Scoring a ragged batch with twenty alternatives a token.
        {"name": "logprob_ragged", "op": "logprob", "train": False, "m": 1000, "v": 50021,
         "d": 5120, "k": 20},
        # Policy training, short micro-batch: log probabilities weighted by
        # advantages and an entropy bonus, with gradients.
        {"name": "logprob_train_short", "op": "logprob", "train": True, "m": 77, "v": 32000,
         "d": 4096, "k": 0},
        # ... full micro-batch and a large vocabulary: the largest case.
        {"name": "logprob_train_full", "op": "logprob", "train": True, "m": 4096, "v": 128000,
         "d": 8192, "k": 0},
        # The norms' weights and gates of 80 layers and the last norm: many small
        # tensors.
        {"name": "adamw_vectors", "op": "adamw", "sizes": "241x8192", "bits": 32, "bf16": False,
         "grad16": False, "copy": False, "scaled": True},
        # fp32 masters of a 7B-sized layer's matrices with the bf16 copies that
        # the next requantization reads.
        {"name": "adamw_layer", "op": "adamw", "sizes": "4x16777216,3x45088768", "bits": 32,
         "bf16": False, "grad16": False, "copy": True, "scaled": True},
        # A bf16 head and embedding, a vocabulary of odd size and odd leftovers,
        # moments in 8 bits.
        {"name": "adamw_bits8", "op": "adamw", "sizes": "2x256107520,3x8191,5x77,1x1", "bits": 8,
         "bf16": True, "grad16": True, "copy": False, "scaled": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the ranges that the listed ones stand for: 1 to 8192 tokens, heads
    of 32 to 256, any vocabulary, 1 to 300 tensors of any size."""
    biggest = max(work(c)["flops"] for c in listed())
    most = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(("rotary", "rotary", "logprob", "adamw"))
        if op == "rotary":
            d = rng.choice((64, 80, 96, 128, 128, 160, 192, 256, 2 * rng.randint(16, 128)))
            hk = _log_int(rng, 1, 32)
            case = {"op": op, "bwd": rng.random() < 0.5, "m": _log_int(rng, 1, 8192),
                    "hq": hk * rng.choice((1, 1, 2, 4, 5, 8)), "hk": hk, "d": d,
                    "rot": rng.choice((d, d, 2 * rng.randint(1, d // 2), d // 4 * 2)),
                    "pairs": rng.choice(("half", "half", "adjacent")),
                    "norm": rng.random() < 0.6, "far": rng.random() < 0.5,
                    "bf16": rng.random() < 0.7, "fused": rng.random() < 0.3}
        elif op == "logprob":
            train = rng.random() < 0.5
            case = {"op": op, "train": train, "m": _log_int(rng, 1, 8192),
                    "v": _log_int(rng, 1000, 128000), "d": _log_int(rng, 1024, 8192) // 8 * 8,
                    "k": 0 if train else rng.choice((0, 1, rng.randint(2, 32)))}
        else:
            sizes = ",".join("%dx%d" % (_log_int(rng, 1, 100), _log_int(rng, 1, 30000000))
                             for _ in range(rng.randint(1, 3)))
            bf16 = rng.random() < 0.4
            case = {"op": op, "sizes": sizes, "bits": rng.choice((8, 32)), "bf16": bf16,
                    "grad16": bf16 or rng.random() < 0.3,
                    "copy": not bf16 and rng.random() < 0.4, "scaled": rng.random() < 0.5}
        w = work(case)
        if w["flops"] <= biggest and w["bytes"] <= most:
            return case


def _sizes(case):
    return [n for part in case["sizes"].split(",")
            for n in [int(part.split("x")[1])] * int(part.split("x")[0])]


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, g, sigma=1.0, dtype=torch.float32):
    return (torch.randn(shape, device="cuda", generator=g) * sigma).to(dtype)


def _frequencies(rot, scaled):
    """Radians a position of each pair, in 64 bits, and the factor of the rotated
    values.  Scaled: four times the trained length of 8192; pairs that turn often
    within it keep their frequency, slow ones are slowed by the factor, with a ramp
    between 32 turns and one."""
    f = [10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)]
    if not scaled:
        return f, 1.0
    factor, trained = 4.0, 8192.0
    keep = [min(1.0, max(0.0, (math.log2(max(trained * v / (2 * math.pi), 1e-30))) / 5.0))
            for v in f]
    return ([v * k + v / factor * (1.0 - k) for v, k in zip(f, keep)],
            0.1 * math.log(factor) + 1.0)


def _prepare_rotary(case, g):
    m, hq, hk, d = case["m"], case["hq"], case["hk"], case["d"]
    dtype = torch.bfloat16 if case["bf16"] else torch.float32
    s = {"op": "rotary", "bwd": case["bwd"], "adjacent": case["pairs"] == "adjacent"}

    def heads(sigma):
        # Some channels of every head are far larger, as after a real projection.
        loud = 1.0 + 4.0 * (torch.rand(d, device="cuda", generator=g) < 0.05)
        if case["fused"]:  # q, k and v side by side in one row
            row = _normal((m, hq + 2 * hk, d), g, sigma) * loud
            row = row.to(dtype)
            return row[:, :hq], row[:, hq:hq + hk]
        return ((_normal((m, hq, d), g, sigma) * loud).to(dtype),
                (_normal((m, hk, d), g, sigma) * loud).to(dtype))

    s["q"], s["k"] = heads(1.5)
    if case["bwd"]:
        s["dq"], s["dk"] = heads(1e-3)
    # Tokens of a packed batch: positions start anew at every sequence, which far
    # ones begin behind a long prefix.
    starts = torch.rand(m, device="cuda", generator=g) < 4.0 / max(m, 4)
    starts[0] = True
    at = torch.arange(m, device="cuda")
    first = torch.where(starts, at, 0).cummax(0).values
    base = torch.randint(0, 131072 if case["far"] else 1, (m,), device="cuda", generator=g)
    s["positions"] = at - first + base[first]
    f, s["factor"] = _frequencies(case["rot"], case["far"])
    s["frequencies"] = torch.tensor(f, dtype=torch.float64, device="cuda")
    # The same as turns a position in units of 2^-64.
    s["turns"] = torch.tensor([int(v / (2 * math.pi) * 2.0 ** 64) for v in f], dtype=torch.int64,
                              device="cuda")
    s["w_q"] = s["w_k"] = None
    if case["norm"]:
        s["w_q"] = 1.0 + _normal((d,), g, 0.1)
        s["w_k"] = 1.0 + _normal((d,), g, 0.1)
    return s


def _prepare_logprob(case, g):
    m, v, d = case["m"], case["v"], case["d"]
    s = {"op": "logprob", "train": case["train"], "k": case["k"]}
    x, w = _normal((m, d), g), _normal((v, d), g, 0.02)
    # Tokens from undecided to sure: the logits' spread doubles and doubles again.
    x *= torch.pow(2.0, torch.randint(0, 3, (m, 1), device="cuda", generator=g).float())
    if not case["train"]:
        # Multiples of 2^-4 and 2^-9: every sum of products is exact in 32 bits,
        # so that ranks do not hang on the order of a sum; equal logits occur.
        x, w = torch.round(x * 16.0) / 16.0, torch.round(w * 512.0) / 512.0
    s["x"], s["w"] = x.to(torch.bfloat16), w.to(torch.bfloat16)
    t = torch.randint(0, v, (m,), device="cuda", generator=g)
    none = torch.rand((m,), device="cuda", generator=g) < 0.1
    s["targets"] = torch.where(none & (torch.arange(m, device="cuda") > 0), IGNORE, t)
    if case["train"]:
        s["dlogp"] = _normal((m,), g, 1.0 / m)
        s["dentropy"] = torch.full((m,), 0.01 / m, device="cuda")
    return s


def _encode(values, mantissa):
    """Codes and scales of non-negative fp32 values in 8 bits, in blocks: a value
    over its block's largest, shifted by 2^-15, as a float of so many mantissa bits
    with its exponent counted from there."""
    shift = 23 - mantissa
    blocks = values.view(-1, BLOCK)
    scales = blocks.amax(1).clamp(min=SMALLEST)
    y = blocks * (1.0 / scales)[:, None] + OFFSET
    u = y.view(torch.int32) - torch.tensor(OFFSET, device=y.device).view(torch.int32)
    u = (u + ((1 << (shift - 1)) - 1) + ((u >> shift) & 1)) >> shift
    return u.view(-1), scales


def _decode(codes, scales, mantissa):
    u = (codes.to(torch.int32) << (23 - mantissa)) + \
        torch.tensor(OFFSET, device=codes.device).view(torch.int32)
    y = u.view(torch.float32) - OFFSET
    return (y.view(-1, BLOCK) * scales[:, None]).view(-1)


def _encode_m(m):
    codes, scales = _encode(m.abs(), 3)
    return torch.where(m < 0, -codes, codes).to(torch.int8), scales


def _encode_v(v):
    r = v.sqrt()
    codes, scales = _encode(r, 4)
    # What is not zero does not become it: it is divided by.
    return torch.where(r > 0, codes.clamp(min=1), codes).to(torch.uint8), scales


def _decode_m(codes, scales):
    mag = _decode(codes.abs(), scales, 3)
    return torch.where(codes < 0, -mag, mag)


def _decode_v(codes, scales):
    return _decode(codes, scales, 4).square()


def _prepare_adamw(case, g):
    sizes = _sizes(case)
    # Parameters and their moments lie in flat buffers, each tensor from a multiple
    # of a block on.
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += (n + BLOCK - 1) // BLOCK * BLOCK
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    for a, n in zip(starts, sizes):
        used[a:a + n] = True
    s = {"op": "adamw", "sizes": sizes, "starts": starts, "bits": case["bits"]}
    # Gradients differ from channel to channel by factors of ten.
    loud = torch.exp(_normal((total // BLOCK, 1), g, 2.0)).expand(-1, BLOCK).reshape(-1)
    grad = _normal((total,), g, 1e-3) * loud
    m = torch.where(used, grad * 0.3 + _normal((total,), g, 2e-4) * loud, 0.0)
    v = torch.where(used, (loud * 1e-3 * (0.5 + torch.rand(total, device="cuda", generator=g)))
                    .square(), 0.0)
    del loud
    grad = grad.to(torch.bfloat16 if case["grad16"] else torch.float32)
    s["grads"] = [grad[a:a + n] for a, n in zip(starts, sizes)]
    s["p"] = _normal((total,), g, 0.02, torch.bfloat16 if case["bf16"] else torch.float32)
    s["copy"] = s["p"].to(torch.bfloat16) if case["copy"] else None
    s["scale"] = torch.full((1,), 0.37, device="cuda") if case["scaled"] else None
    s["step"] = 100
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _encode_m(m)
        s["v"], s["v_scale"] = _encode_v(v)
    else:
        s["m"], s["v"], s["m_scale"], s["v_scale"] = m, v, None, None
    return s


def prepare(case, seed):
    make = {"rotary": _prepare_rotary, "logprob": _prepare_logprob, "adamw": _prepare_adamw}
    return make[case["op"]](case, _generator(seed * 1000 + 7))


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _some(**outs):
    return {k: v for k, v in outs.items() if v is not None}


def _parts(s, flat):
    """A flat buffer's tensors."""
    return [flat[a:a + n] for a, n in zip(s["starts"], s["sizes"])]


def _own(s):
    from aethelstream_amd import loss, optim, rotary
    if s["op"] == "rotary":
        rope = rotary.Rotary(s["turns"], interleaved=s["adjacent"], scale=s["factor"])
        if not s["bwd"]:
            q, k = rotary.apply(s["q"], s["k"], s["positions"], rope, w_q=s["w_q"], w_k=s["w_k"],
                                eps=EPS)
            return {"q": q, "k": k}
        r = rotary.apply_bwd(s["dq"], s["dk"], s["positions"], rope, q=s["q"], k=s["k"],
                             w_q=s["w_q"], w_k=s["w_k"], eps=EPS)
        return _some(dq=r.dq, dk=r.dk, dw_q=r.dw_q, dw_k=r.dw_k)
    if s["op"] == "logprob":
        r = loss.linear_log_probs(s["x"], s["w"], s["targets"], top_k=s["k"], ignore_index=IGNORE)
        out = _some(logp=r.logp, entropy=r.entropy, lse=r.lse, top_logp=r.top_logp,
                    top_ids=r.top_ids)
        if s["train"]:
            out["dx"], out["dw"] = loss.linear_log_probs_bwd(
                s["x"], s["w"], s["targets"], r, s["dlogp"], s["dentropy"], ignore_index=IGNORE)
        return out
    state = optim.AdamWState(s["sizes"], s["m"], s["v"], s["m_scale"], s["v_scale"])
    optim.adamw_step(_parts(s, s["p"]), s["grads"], state, s["step"], lr=LR, betas=BETAS,
                     eps=ADAM_EPS, weight_decay=DECAY, grad_scale=s["scale"],
                     copies=None if s["copy"] is None else _parts(s, s["copy"]))
    m, v = (s["m"], s["v"]) if s["bits"] == 32 else optim.moments(state)
    return _some(p=s["p"], m=m, v=v, copy=s["copy"])


def _plain(s):
    if s["op"] == "rotary":
        return _plain_rotary(s)
    if s["op"] == "logprob":
        return _plain_logprob(s)
    return _plain_adamw(s)


def _turned(x, cos, sin, adjacent):
    """x [M, H, d] with the pairs of its first part rotated."""
    half = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    if adjacent:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    else:
        a, b = x[..., :half], x[..., half:2 * half]
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(2) if adjacent else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_rotary(s):
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()
    dtype = s["q"].dtype
    if not s["bwd"]:
        def forward(x, w):
            x = x.float()
            if w is not None:
                x = x / (x.square().mean(2, keepdim=True) + EPS).sqrt() * w
            return _turned(x, cos, sin, s["adjacent"]).to(dtype)
        return {"q": forward(s["q"], s["w_q"]), "k": forward(s["k"], s["w_k"])}

    def backward(dy, x, w):
        dn = _turned(dy.float(), cos, -sin, s["adjacent"])
        if w is None:
            return dn.to(dtype), None
        x = x.float()
        rms = (x.square().mean(2, keepdim=True) + EPS).sqrt()
        hat, e = x / rms, dn * w
        dx = (e - hat * (e * hat).mean(2, keepdim=True)) / rms
        return dx.to(dtype), (dn * hat).sum((0, 1))

    dq, dw_q = backward(s["dq"], s["q"], s["w_q"])
    dk, dw_k = backward(s["dk"], s["k"], s["w_k"])
    return _some(dq=dq, dk=dk, dw_q=dw_q, dw_k=dw_k)


def _plain_logprob(s):
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    top = z.amax(1)
    total = (z - top[:, None]).exp_().sum(1)
    lse = total.log() + top
    kept = s["targets"] != IGNORE
    at = s["targets"].clamp(min=0)
    hit = z.gather(1, at[:, None])[:, 0]
    logp = torch.where(kept, hit - top - total.log(), 0.0)
    logs = z - lse[:, None]
    entropy = -(logs.exp() * logs).sum(1)
    out = {"logp": logp, "entropy": entropy, "lse": lse}
    if s["k"]:
        # Keys of the values' order, then of the lowest index.
        bits = (z + 0.0).view(torch.int32)
        bits = bits ^ ((bits >> 31) & 0x7fffffff)
        ids = torch.arange(z.shape[1], device=z.device)
        keys = (bits.long() << 32) + (0x7fffffff - ids)
        out["top_ids"] = 0x7fffffff - (keys.topk(s["k"], dim=1).values & 0xffffffff)
        out["top_logp"] = logs.gather(1, out["top_ids"])
    if s["train"]:
        del z
        a = torch.where(kept, s["dlogp"], 0.0)[:, None]
        g = -logs.exp() * (a + s["dentropy"][:, None] * (logs + entropy[:, None]))
        rows = torch.arange(g.shape[0], device=g.device)
        g[rows, at] += a[:, 0]
        out["dx"] = (g @ w).to(torch.bfloat16)
        out["dw"] = (g.t() @ x).to(torch.bfloat16)
    return out


def _plain_adamw(s):
    b1, b2 = BETAS
    keep = 1.0 - LR * DECAY
    size = LR / (1.0 - b1 ** s["step"])
    inv = 1.0 / math.sqrt(1.0 - b2 ** s["step"])
    bits8 = s["bits"] == 8
    if bits8:
        m_all, v_all = _decode_m(s["m"], s["m_scale"]), _decode_v(s["v"], s["v_scale"])
    else:
        m_all, v_all = s["m"], s["v"]

    def update(p, grad, m, v, copy):
        grad = grad.float()
        if s["scale"] is not None:
            grad = grad * s["scale"]
        m.mul_(b1).add_(grad * (1.0 - b1))
        v.mul_(b2).add_(grad * grad * (1.0 - b2))
        new = p.float() * keep - m / (v.sqrt() * inv + ADAM_EPS) * size
        p.copy_(new)
        if copy is not None:
            copy.copy_(new)

    copies = [None] * len(s["sizes"]) if s["copy"] is None else _parts(s, s["copy"])
    list(map(update, _parts(s, s["p"]), s["grads"], _parts(s, m_all), _parts(s, v_all), copies))
    if bits8:
        codes, scales = _encode_m(m_all)
        s["m"].copy_(codes), s["m_scale"].copy_(scales)
        codes, scales = _encode_v(v_all)
        s["v"].copy_(codes), s["v_scale"].copy_(scales)
        m_all, v_all = _decode_m(s["m"], s["m_scale"]), _decode_v(s["v"], s["v_scale"])
    return _some(p=s["p"], m=m_all, v=v_all, copy=s["copy"])


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    if case["op"] == "rotary":
        n = case["m"] * (case["hq"] + case["hk"]) * case["d"]
        size = 2 if case["bf16"] else 4
        moved = 2 + (case["bwd"] and case["norm"])  # in and out, and x in the norms' backward
        vectors = 4 * case["rot"] + 8 * case["m"] + 8 * case["d"] * case["norm"]
        return {"bytes": moved * size * n + vectors,
                "flops": (3 + 4 * case["norm"] + 6 * (case["bwd"] and case["norm"])) * n}
    if case["op"] == "logprob":
        m, v, d = case["m"], case["v"], case["d"]
        # x, W and targets in, three values a token and the alternatives out.
        moved = 2 * (m + v) * d + 20 * m + 12 * m * case["k"]
        if not case["train"]:
            return {"bytes": moved, "flops": 2 * m * v * d}
        # The logits again (they are not kept), dx and dW.
        return {"bytes": moved + 2 * (m + v) * d + 8 * m, "flops": 8 * m * v * d}
    n = sum(_sizes(case))
    p = 2 if case["bf16"] else 4
    g = 2 if case["grad16"] else 4
    # p, m and v in and out, the gradient in; what 8-bit moments stand for out.
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8
    return {"bytes": int((2 * p + g + state + 2 * case["copy"]) * n), "flops": 16 * n}


# --------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "logprob": _exact_logprob, "adamw": _exact_adamw}[s["op"]](s)


def _exact_rotary(s):
    half = s["frequencies"].shape[0]
    d = s["q"].shape[2]
    angle = torch.outer(s["positions"].double(), s["frequencies"])
    unit = torch.polar(torch.full_like(angle, s["factor"]), angle).unsqueeze(1)
    # The places of each pair's two values.
    i = torch.arange(half, device=angle.device)
    first, second = (2 * i, 2 * i + 1) if s["adjacent"] else (i, i + half)

    def rotate(x, by):
        y = x.clone()
        z = torch.complex(x[..., first], x[..., second]) * by
        y[..., first], y[..., second] = z.real, z.imag
        return y

    def norm(x):
        return torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS)

    if not s["bwd"]:
        out = {}
        for name in ("q", "k"):
            x, w = s[name].double(), s["w_" + name]
            out[name] = rotate(x if w is None else x / norm(x) * w.double(), unit)
        return out
    out = {}
    for name in ("q", "k"):
        x, w = s[name].double(), s["w_" + name]
        dn = rotate(s["d" + name].double(), unit.conj())
        if w is not None:
            rms = norm(x)
            out["dw_" + name] = (dn * x / rms).sum(dim=(0, 1))
            dhat = dn * w.double()
            dn = dhat / rms - x * (dhat * x).sum(-1, keepdim=True) / (d * rms ** 3)
        out["d" + name] = dn
    return out


def _exact_logprob(s):
    x, w, t = s["x"].double(), s["w"].double(), s["targets"]
    z = torch.matmul(x, w.t())
    lse = torch.logsumexp(z, 1)
    kept = t != IGNORE
    at = torch.where(kept, t, 0).unsqueeze(1)
    logp = torch.where(kept, torch.gather(z, 1, at).squeeze(1) - lse, torch.zeros_like(lse))
    p = torch.softmax(z, 1)
    entropy = lse - (p * z).sum(1)
    out = {"logp": logp, "entropy": entropy, "lse": lse}
    if s["k"]:
        values, ids = torch.sort(z, dim=1, descending=True, stable=True)
        out["top_ids"] = ids[:, :s["k"]].contiguous()
        out["top_logp"] = values[:, :s["k"]] - lse.unsqueeze(1)
    if s["train"]:
        a = torch.where(kept, s["dlogp"].double(), torch.zeros_like(lse)).unsqueeze(1)
        h = s["dentropy"].double().unsqueeze(1)
        # d entropy / d z = -p (log p + entropy)
        z = -p * (a + h * (z - lse.unsqueeze(1) + entropy.unsqueeze(1)))
        del p
        z.scatter_add_(1, at, a)
        out["dx"], out["dw"] = torch.matmul(z, w), torch.matmul(z.t(), x)
    return out


def _exact_adamw(s):
    b1, b2 = BETAS
    t = s["step"]

    def code(y, mantissa):
        """The nearest value of the form that 8 bits hold, of y in [0, 1]."""
        y = y + OFFSET
        unit = torch.exp2(torch.floor(torch.log2(y)) - mantissa)
        return torch.round(y / unit) * unit - OFFSET

    bits8 = s["bits"] == 8
    if bits8:
        m, v = _decode_m(s["m"], s["m_scale"]).double(), _decode_v(s["v"], s["v_scale"]).double()
    else:
        m, v = s["m"].double(), s["v"].double()
    # The blocks' gaps hold zeros and keep them; what p holds there stays.
    grad = torch.zeros_like(m)
    used = torch.zeros_like(m, dtype=torch.bool)
    for a, n, g in zip(s["starts"], s["sizes"], s["grads"]):
        grad[a:a + n] = g.double()
        used[a:a + n] = True
    if s["scale"] is not None:
        grad = grad * s["scale"].double()
    m = m * b1 + grad * (1 - b1)
    v = v * b2 + grad ** 2 * (1 - b2)
    del grad
    p = s["p"].double()
    new = p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + ADAM_EPS)
    p = torch.where(used, new, p)
    copy = None if s["copy"] is None else torch.where(used, new, s["copy"].double())
    if bits8:
        blocks = m.view(-1, BLOCK)
        top = blocks.abs().amax(1, keepdim=True).clamp(min=SMALLEST)
        m = (torch.sign(blocks) * code(blocks.abs() / top, 3) * top).view(-1)
        blocks = torch.sqrt(v).view(-1, BLOCK)
        top = blocks.amax(1, keepdim=True).clamp(min=SMALLEST)
        least = torch.where(blocks > 0, OFFSET * 2.0 ** -4, 0.0)
        v = (torch.maximum(code(blocks / top, 4), least) * top).square().view(-1)
    return _some(p=p, m=m, v=v, copy=copy)
